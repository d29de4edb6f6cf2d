// Tiles of C = A B^T on the matrix cores, both operands stored with the reduction index contiguous, staged through LDS by DMA.
//
// A stage holds RB bytes of every row of the tile (BM rows of A, BN rows of B).  One DMA instruction of a wave lands 1 KB lane-linear in LDS, so the
// 16-byte XOR swizzle that spreads a fragment read over all banks is applied to the per-lane SOURCE address and again on the read: LDS row r
// holds source chunk (slot ^ key(r)).  ST buffers form a ring.  A stage is two (four) steps; the fragments of each are read while the MFMAs of the one before
// run.  The one barrier of a stage stands in front of its last step, when its last fragments are in registers: behind it the buffer takes the requests of stage
// s + ST, and stage s + 1, whose requests every wave has waited for with a counted vmcnt, is read.
//
// Operand rows beyond the matrix are clamped to its last row: they are read, multiplied and never stored.  The reduction length is a whole number of
// stages; what lies behind the real end of a row is zero in memory.
#pragma once
#include "common.h"

namespace saunet {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

// lane-linear 1 KB from (uniform base + per-lane byte offset) to LDS address lds_dst; M0 is restored for the compiler's own use
__device__ __forceinline__ void nt_dma16(const char* sbase, unsigned voff, unsigned lds_dst)
{
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds_dst) : "memory");
}
__device__ __forceinline__ const char* nt_uniform(const char* p)
{
    const unsigned long long u = (unsigned long long)p;
    return (const char*)(((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)u));
}
// all LDS reads of this wave have returned and at most N of its DMA requests are in flight, then the workgroup barrier
template <int N> __device__ __forceinline__ void nt_wait_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(N) : "memory");
}

// Workgroup ids go round the eight XCDs, each with an L2 of its own: XCD x takes the x-th eighth of the work, so that neighbours share an L2
__device__ __forceinline__ int nt_xcd(int id, int total)
{
    const int x = id & 7, q = total >> 3, rest = total & 7;
    return x * q + (x < rest ? x : rest) + (id >> 3);
}
// t-th tile of a rows x cols grid walked in bands of eight tile rows: the tiles in flight share both operands
__device__ __forceinline__ void nt_band(int t, int rows, int cols, int& r, int& c)
{
    const int band = t / (8 * cols), h = rows - band * 8 < 8 ? rows - band * 8 : 8, in = t - band * 8 * cols;
    r = band * 8 + in % h;
    c = in / h;
}

// float16 pairs: a row is a sequence of blocks of 32 elements, each 64 bytes of high parts followed by 64 bytes of low parts.  Two
// significands of 11 bits and the sign of lo are 23 bits: x = hi + lo to 2^-23 of x (a quarter of the float32 numbers in [1, 2) are off by more than 2^-24).
// hi hi + hi lo + lo hi in float32; |lo| <= 2^-11 |x|, so what is dropped, lo lo, is up to 2^-22 of |a| |b|.
struct NtF16Pair {
    // the MFMA's adder cuts off instead of rounding, which over a long sum of one sign is a bias: 256 additions cost 6e-6 of the sum.  Every FLUSH stages the
    // accumulators are added to a float32 total and start again.
    static constexpr int RB = 128, KSUB = 2, PARTS = 2, FLUSH = 8;
    typedef f32x16 Acc;
    static __device__ __forceinline__ int chunk(int ks, int part, int half) { return part * 4 + ks * 2 + half; }
    static __device__ __forceinline__ void mma(const u32x4 (&a)[2], const u32x4 (&b)[2], Acc& c)
    {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a[1]), __builtin_bit_cast(f16x8_t, b[0]), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a[0]), __builtin_bit_cast(f16x8_t, b[1]), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a[0]), __builtin_bit_cast(f16x8_t, b[0]), c, 0, 0, 0);
    }
};
// two such blocks a stage: half the barriers
struct NtF16Pair2 : NtF16Pair {
    static constexpr int RB = 256, KSUB = 4, FLUSH = 4;
    static __device__ __forceinline__ int chunk(int ks, int part, int half) { return (ks >> 1) * 8 + part * 4 + (ks & 1) * 2 + half; }
};
// int8, 64 elements a stage
struct NtI8 {
    static constexpr int RB = 64, KSUB = 2, PARTS = 1, FLUSH = 0;          // integer sums are exact
    typedef i32x16 Acc;
    static __device__ __forceinline__ int chunk(int ks, int, int half) { return ks * 2 + half; }
    static __device__ __forceinline__ void mma(const u32x4 (&a)[1], const u32x4 (&b)[1], Acc& c)
    {
        c = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a[0]), __builtin_bit_cast(i32x4, b[0]), c, 0, 0, 0);
    }
};

// BM x BN tile by WGM x WGN waves; wave (wm, wn) owns TM x TN blocks of 32 x 32.  KW > 1: KW such sets of waves, each of which takes a KW-th of every
// stage and ends with a sum of its own; the caller adds them.  Accumulator element r of lane l: row 8 (r / 4) + 4 (l / 32) + r % 4
// (operand A), column l % 32 (operand B).
template <class Op, int BM_, int BN_, int WGM_, int WGN_, int ST_, int KW_ = 1> struct NtCore {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, ST = ST_, KW = KW_, RB = Op::RB, MY = Op::KSUB / KW;          // MY: steps of a stage that are a wave's
    static constexpr int NW = WGM * WGN * KW, NT = NW * 64, TM = BM / WGM / 32, TN = BN / WGN / 32;
    static constexpr int STAGE = (BM + BN) * RB, LDS = ST * STAGE, CPR = RB / 16, RPI = 1024 / RB;
    static constexpr int QA = BM * RB / 1024 / NW, QB = BN * RB / 1024 / NW, LPW = QA + QB;
    static_assert(QA * NW * 1024 == BM * RB && QB * NW * 1024 == BN * RB, "every wave requests whole instructions of one operand");
    static_assert(ST >= 2 && ST <= 8 && (ST - 1) * LPW < 64 && (MY == 1 || MY == 2 || MY == 4), "vmcnt counts to 63");
    typedef typename Op::Acc Acc;

    // 256 bytes of LDS answer at once: 1 (2, 4) rows of the tile beside each other, so rows that agree modulo 1 (2, 4) have to differ in their key
    static __device__ __forceinline__ int key(int row) { return CPR == 16 ? (row & 15) : CPR == 8 ? ((row >> 1) & 7) : ((row >> 2) & 3); }

    // a, b: first byte of the tile's first row at its first stage (uniform); arows, brows: rows that exist from there on (>= 1)
    static __device__ __forceinline__ void run(const char* a, unsigned lda, int arows, const char* b, unsigned ldb, int brows, int ksteps, unsigned char* smem,
                                               Acc (&total)[TM][TN])
    {
        a = nt_uniform(a); b = nt_uniform(b);
        ksteps = __builtin_amdgcn_readfirstlane(ksteps);
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wk = wave / (WGM * WGN), wm = wave / WGN % WGM, wn = wave % WGN;
        const unsigned lds0 = (unsigned)(uintptr_t)smem;
        unsigned voff[LPW];
#pragma unroll
        for (int q = 0; q < LPW; ++q) {
            const bool isa = q < QA;
            const int row = ((isa ? q : q - QA) * NW + wave) * RPI + lane / CPR;
            const int rows = isa ? arows : brows;
            voff[q] = (unsigned)(row < rows ? row : rows - 1) * (isa ? lda : ldb) + (unsigned)(((lane % CPR) ^ key(row)) * 16);
        }
        auto issue = [&](int s) {
            const unsigned dst = lds0 + (unsigned)(s % ST) * STAGE;
            const char* pa = a + (long)s * RB;
            const char* pb = b + (long)s * RB;
#pragma unroll
            for (int q = 0; q < LPW; ++q)
                nt_dma16(q < QA ? pa : pb, voff[q], dst + (q < QA ? q * NW + wave : BM * RB / 1024 + (q - QA) * NW + wave) * 1024);
        };
        const int r0 = lane & 31, half = lane >> 5, k0 = key(r0);
        u32x4 fa[2][TM][Op::PARTS], fb[2][TN][Op::PARTS];
        Acc part[TM][TN] = {};
        Acc (&acc)[TM][TN] = Op::FLUSH ? part : total;
        // step ks of stage s into fragments f
        auto read = [&](int s, int ks, int f) {
            const unsigned char* st = smem + (s % ST) * STAGE;
            const unsigned char* sa = st + (wm * (BM / WGM) + r0) * RB;
            const unsigned char* sb = st + BM * RB + (wn * (BN / WGN) + r0) * RB;
#pragma unroll
            for (int p = 0; p < Op::PARTS; ++p) {
                const int at = (Op::chunk(KW > 1 ? wk * MY + ks : ks, p, half) ^ k0) * 16;
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[f][i][p] = *(const u32x4*)(sa + i * 32 * RB + at);
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[f][j][p] = *(const u32x4*)(sb + j * 32 * RB + at);
            }
        };
        auto mma = [&](int f) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) Op::mma(fa[f][i], fb[f][j], acc[i][j]);
        };
        // this wave's LDS reads are in registers, its requests of all but the newest `young` stages have landed; then the workgroup's have
        auto settle = [&](int young) {
            switch (young) {
            case 0: nt_wait_barrier<0>(); break;
            case 1: nt_wait_barrier<LPW>(); break;
            case 2: nt_wait_barrier<(ST > 2 ? 2 : 0) * LPW>(); break;
            case 3: nt_wait_barrier<(ST > 3 ? 3 : 0) * LPW>(); break;
            case 4: nt_wait_barrier<(ST > 4 ? 4 : 0) * LPW>(); break;
            case 5: nt_wait_barrier<(ST > 5 ? 5 : 0) * LPW>(); break;
            case 6: nt_wait_barrier<(ST > 6 ? 6 : 0) * LPW>(); break;
            default: nt_wait_barrier<(ST > 7 ? 7 : 0) * LPW>(); break;
            }
        };
        for (int s = 0; s < ST && s < ksteps; ++s) issue(s);
        settle((ksteps < ST ? ksteps : ST) - 1);
        read(0, 0, 0);
        auto stage = [&](int s, int odd) {                                              // odd: the fragments that hold its first step
#pragma unroll
            for (int ks = 0; ks + 1 < MY; ++ks) {
                read(s, ks + 1, (ks + 1) & 1);
                __builtin_amdgcn_sched_barrier(0);
                mma(ks & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (s + 1 < ksteps) {
                settle(ksteps - 2 - s < ST - 2 ? ksteps - 2 - s : ST - 2);          // stage s + 1 is there; nobody reads stage s any more
                if (s + ST < ksteps) issue(s + ST);
                read(s + 1, 0, MY == 1 ? odd ^ 1 : 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            mma(MY == 1 ? odd : 1);
            __builtin_amdgcn_sched_barrier(0);
            if (Op::FLUSH && ((s & (Op::FLUSH - 1)) == Op::FLUSH - 1 || s + 1 == ksteps)) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) { total[i][j] += part[i][j]; part[i][j] = Acc{}; }
            }
        };
        if constexpr (MY == 1) {
            for (int s = 0; s < ksteps; s += 2) { stage(s, 0); if (s + 1 < ksteps) stage(s + 1, 1); }
        } else {
            for (int s = 0; s < ksteps; ++s) stage(s, 0);
        }
    }
};

}  // namespace saunet
