// Newton-Schulz orthogonalisation of a list of matrices and the Muon step around it.
//
//   X0 = G / max(|G|_F, eps);   S = X X^T,  X <- (a I + b S + c S^2) X,  `steps` times          (rows <= columns; the transpose otherwise)
//
// One call takes any number of matrices of any shapes: every launch below covers one phase of ALL of them, a workgroup finds its matrix in a
// table of tile prefixes.  The chain is some twenty launches for five steps whatever the list is, and one more behind each launch that cuts tiles (4096 x 4096:
// 34 in all); two chains where newton_schulz gets both short and long matrices.
//
// Composition.  S_k+1 = P_k S_k P_k with P_k = a I + b S_k + c S_k^2, and all of them commute, so some steps run on the m x m matrices alone (S and
// the product of the P_k) before X is touched: three, then two at a time; 6 m^2 n + 14 m^3 operations for five steps against 5 (3 m^2 n + m^3).  Equal for
// a square, 2.4x less at n = 27 m.  What it costs in digits: an error of S grows by a^2 = 12 with every step it is carried through, and the product is
// kept as (P_2 P_1 P_0 - a^3 I), up to 41 in size where s is near 1, for a result near 1.  In the first block the s^2 add up to 1, so the 41 are divided by
// sqrt(m): three from m = 256 on, two before.  Later most s are near 1, so there P is kept as (a - 1) I + b S + c S^2, near zero, and two steps are composed.
// newton_schulz takes matrices of up to 128 rows step by step, in a chain of their own.  Distance from float64 over that of the same chain in float32
// matrices, gradient-like input, five steps: 0.6 - 1.2 for 33 .. 128 rows (three + two: 1.4 - 4.6), 0.9 - 1.1 for 129 .. 255 (three + two: 1.2 - 3.8), 1.2 at
// 300, 0.8 at 512, 0.4 at 1000 and above.
// A Muon step whose list holds a matrix of more than 128 rows takes ALL its matrices of more than 32 through one chain of three + two, at the distances in
// brackets (33 x 40 3.9, 64 x 576 1.5, 128 x 736 1.1; two + two + one: 1.4, 0.6, 0.6): there the update is multiplied by the rate and added to a rounded
// parameter.  SAUNet's step 936 us; with two + two + one 1112, in two chains 1090.
//
// Number format.  Every matrix between the first and the last pass is a pair of float16 planes, x = hi + lo to 2^-23 (nt_tiles.h: 128-byte blocks of 32
// elements), scaled by a power of two that the host derives from the singular values' range.  A product is then three float16 MFMAs with float32
// accumulation, at a sixth of the cost of the float32 MFMA; its operands and the dropped low parts can cost four times float32's half steps, measured the whole
// chain is about as far from float64 as the float32 one (above).  Products of symmetric matrices compute the lower tiles only and write both halves.
// X and X^T are both kept: each is the operand with the contiguous reduction index in one of the two rectangular products.
#include "nt_tiles.h"
#include <algorithm>

namespace saunet {

struct NsSplit { int p, full, s, c; };    // first workgroup, tiles done whole, parts of each of the others, first of those others in the finishing launch
enum { NS_GRAM = 0, NS_ONE, NS_TWO, NS_KINDS };
struct NsItem {            // one matrix, as the host lays it out
    const void* src; void* dst; float* buf; char* ws;
    int ld_src, ld_dst, rows, cols;
    int p_norm, p_pack, p_app;       // index of the matrix's first workgroup in the launches of each kind
    NsSplit split[NS_KINDS];
    // (number by number: an index that the compiler does not know, or a choice between whole structures, puts them into scratch memory: 2 - 3 us a launch)
    __device__ __forceinline__ NsSplit of(int kind) const
    {
        const bool g = kind == NS_GRAM, o = kind == NS_ONE;
        const NsSplit x = split[NS_GRAM], y = split[NS_ONE], z = split[NS_TWO];
        return NsSplit{g ? x.p : o ? y.p : z.p, g ? x.full : o ? y.full : z.full, g ? x.s : o ? y.s : z.s, g ? x.c : o ? y.c : z.c};
    }
};
constexpr int NS_CHUNK = 36;                 // of them are kernel arguments
struct NsItems { NsItem it[NS_CHUNK]; };
static_assert(sizeof(NsItems) <= 4064, "kernel arguments end at 4 KB");
constexpr int NS_NORM = 4096;                // elements a workgroup of the norm pass takes

enum { NS_X = -1, NS_A = 0, NS_P, NS_R, NS_Q0, NS_Q1, NS_NSYM };
struct NsView {
    int m, n, mp, np, tall;
    char *x, *s0; float* t0; long bx, bs;
    static long bytes(int rows, int cols)
    {
        const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows, mp = (m + 63) / 64 * 64, np = (n + 63) / 64 * 64;
        return 256 + 3 * mp * np * 4 + NS_NSYM * mp * mp * 4;
    }
    __device__ explicit NsView(const NsItem& it)
    {
        tall = it.rows > it.cols;
        m = tall ? it.cols : it.rows; n = tall ? it.rows : it.cols;
        mp = (m + 63) / 64 * 64; np = (n + 63) / 64 * 64;
        bx = (long)mp * np * 4; bs = (long)mp * mp * 4;
        t0 = (float*)it.ws; x = it.ws + 256; s0 = x + 3 * bx;
    }
    __device__ __forceinline__ char* xt(int i) const { return x + (1 + i) * bx; }
    __device__ __forceinline__ char* sym(int i) const { return s0 + i * bs; }
    __device__ __forceinline__ float* part() const { return (float*)(s0 + NS_NSYM * bs); }
    // A matrix whose norm is below eps is kept as X / t, so that its elements do not sink below what a float16 pair resolves (norm = 1e-6 eps, 300 x 500: 4e-4 of
    // the result before, 1e-7 now).  t starts as the power of two t0 >= norm / eps and grows with every application of a polynomial by a power of two that
    // bounds its growth, up to 1; `grown` is the product of those bounds.  All other matrices have t0 = 1, for which nothing below changes a bit.
    __device__ __forceinline__ float t(float grown) const { const float v = *t0 * grown; return v < 1.f ? v : 1.f; }
};

// the matrix whose workgroups include `id`: the last whose first(i) is not above it; two rounds of one load a lane (count <= 4096)
template <typename F> __device__ __forceinline__ int ns_find(int count, int id, F first)
{
    const int lane = threadIdx.x & 63, step = (count + 63) >> 6;
    int base = 0;
    if (step > 1) {
        const int i = lane * step;
        base = (__popcll(__ballot(i < count && first(i < count ? i : 0) <= id)) - 1) * step;
    }
    const int i = base + lane;
    return __builtin_amdgcn_readfirstlane(base + __popcll(__ballot((step == 1 || lane < step) && i < count && first(i < count ? i : 0) <= id)) - 1);
}

// A single matrix is a kernel argument (the table of others is two loads one after the other in front of every tile) and needs no set-up launch:
// 512 x 13824 310 -> 303 us a call
struct NsTable { const NsItem* all; int count; NsItem one; };
template <typename F> __device__ __forceinline__ NsItem ns_item(const NsTable& t, int id, F first)
{
    if (t.count == 1) return t.one;
    return t.all[ns_find(t.count, id, [&](int i) { return first(t.all[i]); })];
}

__global__ void ns_setup_kernel(NsItems items, int count, NsItem* __restrict__ tab)
{
    if ((int)threadIdx.x < count) tab[threadIdx.x] = items.it[threadIdx.x];
}

// ---- element access -------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float ns_load(const T* p);
template <> __device__ __forceinline__ float ns_load<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ns_load<u16>(const u16* p) { return Elem<u16>::load(p); }
template <> __device__ __forceinline__ float ns_load<_Float16>(const _Float16* p) { return (float)*p; }
template <typename T> __device__ __forceinline__ void ns_store(T* p, float v);
template <> __device__ __forceinline__ void ns_store<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void ns_store<u16>(u16* p, float v) { Elem<u16>::store(p, v); }
template <> __device__ __forceinline__ void ns_store<_Float16>(_Float16* p, float v) { *p = (_Float16)v; }

struct Pair { _Float16 h, l; };
__device__ __forceinline__ Pair ns_split(float v) { Pair s; s.h = (_Float16)v; s.l = (_Float16)(v - (float)s.h); return s; }

// hyper (Muon): [0] lr [1] momentum [2] weight_decay [3] nesterov [4] grad_scale
// buf <- momentum buf + (1 - momentum) g;  the matrix to orthogonalise is (1 - momentum) g + momentum buf with nesterov, buf without.  buf is the
// NEW buffer in ns_update, which the norm pass and the pack pass both evaluate.
__device__ __forceinline__ float ns_momentum(float g, float buf, const float* h) { const float gs = g * h[4]; return fmaf(h[1], buf - gs, gs); }
__device__ __forceinline__ float ns_update(float g, float buf, const float* h) { const float gs = g * h[4]; return h[3] != 0.f ? fmaf(h[1], buf - gs, gs) : buf; }

// ---- sums of squares (and the momentum update): float64 partials of NS_NORM elements each, summed in index order by the pack pass ------------
template <typename T, bool MUON> __global__ __launch_bounds__(256) void ns_norm_kernel(NsTable tab, const float* __restrict__ hyper, double* __restrict__ part)
{
    __shared__ double s_sum[4];
    const int id = blockIdx.x;
    const NsItem it = ns_item(tab, id, [&](const NsItem& t) { return t.p_norm; });
    const long total = (long)it.rows * it.cols, e0 = (long)(id - it.p_norm) * NS_NORM;
    float h[5] = {0.f, 0.f, 0.f, 0.f, 1.f};
    if (MUON) for (int i = 0; i < 5; ++i) h[i] = hyper[i];
    double sum = 0.0;
    constexpr int EACH = NS_NORM / 256;
    float g[EACH], old[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const long e = e0 + k * 256 + threadIdx.x;
        const long r = it.ld_src == it.cols ? 0 : e / it.cols;
        g[k] = old[k] = 0.f;
        if (e < total) { g[k] = ns_load((const T*)it.src + (r * (it.ld_src - it.cols) + e)); if (MUON) old[k] = it.buf[e]; }
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const long e = e0 + k * 256 + threadIdx.x;
        if (e >= total) break;
        float u = g[k];
        if (MUON) { const float b = ns_momentum(g[k], old[k], h); it.buf[e] = b; u = ns_update(g[k], b, h); }
        sum += (double)u * (double)u;
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[id] = ((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3];
}

// ---- X0 and X0^T as scaled float16 pairs: a workgroup takes 64 x 64 elements --------------------------------------------------------
template <typename T, bool MUON> __global__ __launch_bounds__(256) void ns_pack_kernel(NsTable tab, const float* __restrict__ hyper, const double* __restrict__ part, float eps, float sx)
{
    __shared__ float s_t[64][65];
    __shared__ double s_sum[4];
    const int tid = threadIdx.x, id = blockIdx.x;
    const NsItem it = ns_item(tab, id, [&](const NsItem& t) { return t.p_pack; });
    const NsView v(it);
    float h[5] = {0.f, 0.f, 0.f, 0.f, 1.f};
    if (MUON) for (int i = 0; i < 5; ++i) h[i] = hyper[i];
    // tiles in the caller's orientation: r along its rows, c along its columns; the elements are on their way while the norm is summed
    const int rp = v.tall ? v.np : v.mp, cp = v.tall ? v.mp : v.np, tc = (cp + 63) / 64, t = id - it.p_pack;
    const int r0 = t / tc * 64, c0 = t % tc * 64;
    float g[16], buf[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int r = r0 + k * 4 + (tid >> 6), c = c0 + (tid & 63);
        g[k] = buf[k] = 0.f;
        if (r < it.rows && c < it.cols) { g[k] = ns_load((const T*)it.src + (long)r * it.ld_src + c); if (MUON) buf[k] = it.buf[(long)r * it.cols + c]; }
    }
    const int nblk = (int)(((long)it.rows * it.cols + NS_NORM - 1) / NS_NORM);
    double sum = 0.0;
    for (int i = tid; i < nblk; i += 256) sum += part[it.p_norm + i];
    sum = wave_sum(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    const double norm = sqrt(((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3]);
    // (a NaN norm stays NaN)
    double t0 = 1.0;
    if (norm < (double)eps && norm > 0.0) { t0 = ldexp(1.0, (int)ceil(log2(norm / (double)eps))); t0 = t0 < 0x1p-126 ? 0x1p-126 : t0; }
    if (id == it.p_pack && tid == 0) *v.t0 = (float)t0;
    const double inv = (double)sx / ((norm <= (double)eps ? (double)eps : norm) * t0);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        // (a padding element is zero, not zero times a scale that may be NaN)
        const int r = r0 + k * 4 + (tid >> 6), c = c0 + (tid & 63);
        s_t[k * 4 + (tid >> 6)][tid & 63] = r < it.rows && c < it.cols ? (float)((double)(MUON ? ns_update(g[k], buf[k], h) : g[k]) * inv) : 0.f;
    }
    __syncthreads();
    // 8 consecutive elements a thread: 16 bytes of high and of low parts; along[] runs along the caller's rows, across[] along its columns
    char* along = v.tall ? v.xt(0) : v.x;
    char* across = v.tall ? v.x : v.xt(0);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        for (int k = tid; k < 64 * 8; k += 256) {
            const int o = k >> 3, e = (k & 7) * 8;                    // line of the destination, element in it
            const int row = (side ? c0 : r0) + o, col = (side ? r0 : c0) + e;
            if (row >= (side ? cp : rp) || col >= (side ? rp : cp)) continue;
            f16x8_t hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) { const Pair s = ns_split(side ? s_t[e + i][o] : s_t[o][e + i]); hi[i] = s.h; lo[i] = s.l; }
            char* d = (side ? across : along) + (long)row * (side ? rp : cp) * 4 + (col >> 5) * 128 + (col & 31) * 2;
            *(f16x8_t*)d = hi; *(f16x8_t*)(d + 64) = lo;
        }
    }
}

// ---- products -----------------------------------------------------------------------------------------------------------------------
// 64 KB of LDS, two workgroups a CU.  (Twice the stages in one workgroup a CU brought nothing, also where a launch has fewer workgroups than CUs.)  The
// small tile takes 64 elements a stage: half the barriers, 13.6 -> 11.5 us a launch at 512 rows, 19.2 -> 18.1 over SAUNet's list; matrices are padded to
// 64 for it.
typedef NtCore<NtF16Pair, 128, 128, 2, 2, 2> NsCore128;
typedef NtCore<NtF16Pair2, 64, 64, 2, 2, 2> NsCore64;
typedef NtCore<NtF16Pair, 128, 128, 4, 2, 2> NsCore128W;         // eight waves, for launches without a second workgroup for every CU (six 1000 x 1024 matrices 755 -> 701 us, the same with two sets of four waves that
                                                                 // share the reduction; 4096 x 4096 with it throughout 4219 -> 4699)
typedef NtCore<NtF16Pair2, 32, 32, 1, 1, 4, 4> NsCore32;           // four waves share one reduction; never cut
constexpr int NS_SLOTS = 512;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

// Accumulator quad b of a thread: the four rows i .. i + 3 of column j, relative to the tile
template <class Core> struct NsQuads {
    static constexpr int N = Core::TM * Core::TN * 4 / Core::KW, FLOATS = Core::BM * Core::BN;          // (of a shared reduction a wave keeps group `wave`)
    static __device__ __forceinline__ int group(int b) { return Core::KW > 1 ? (int)threadIdx.x >> 6 : b & 3; }
    static __device__ __forceinline__ void at(int b, int& i, int& j)
    {
        const int lane = threadIdx.x & 63, wave = Core::KW > 1 ? 0 : threadIdx.x >> 6, ti = b / (4 * Core::TN), tj = b / 4 % Core::TN, g = group(b);
        i = (wave / Core::WGN) * (Core::BM / Core::WGM) + ti * 32 + g * 8 + (lane >> 5) * 4;
        j = (wave % Core::WGN) * (Core::BN / Core::WGN) + tj * 32 + (lane & 31);
    }
    template <typename F> static __device__ __forceinline__ void each(F f)
    {
#pragma unroll
        for (int b = 0; b < N; ++b) { int i, j; at(b, i, j); f(b, i, j); }
    }
    static __device__ __forceinline__ void quad(const f32x16 (&acc)[Core::TM][Core::TN], int b, float (&q)[4])
    {
#pragma unroll
        for (int r = 0; r < 4; ++r) q[r] = acc[b / (4 * Core::TN)][b / 4 % Core::TN][(b & 3) * 4 + r];
    }
};
// four consecutive elements (row j, columns i .. i + 3) of a pair matrix with ldb bytes a row
__device__ __forceinline__ void ns_read4(const char* p, long ldb, int j, int i, float (&v)[4])
{
    const char* s = p + (long)j * ldb + (i >> 5) * 128 + (i & 31) * 2;
    const f16x4_t h = *(const f16x4_t*)s, l = *(const f16x4_t*)(s + 64);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (float)h[r] + (float)l[r];
}
__device__ __forceinline__ void ns_split4(const float (&v)[4], f16x4_t& h, f16x4_t& l)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) { const Pair s = ns_split(v[r]); h[r] = s.h; l[r] = s.l; }
}
// (i .. i + 3, j) of a tile of a symmetric matrix that lies on the diagonal: the part above it is dropped and the part below written to both halves, so
// that the stored matrix is symmetric to the last bit.  An antisymmetric rounding error would not shrink with a I + P as the error of S does: it grew
// six-fold a product (2e-5 of |X| after five steps).  put(row, col, pair)
template <typename F> __device__ __forceinline__ void ns_both_halves(int i, int j, const float (&v)[4], F put)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (i + r < j) continue;
        const Pair s = ns_split(v[r]);
        put(j, i + r, s);
        put(i + r, j, s);
    }
}

// A tile of pairs in LDS, between the accumulators and memory: rows of BM pairs, the 16-byte chunks of row r swapped by XOR with r so that a column of
// them is spread over the banks.  Straight from the accumulators a store is 8 bytes in each of 32 rows, or 2 bytes in a row: such an epilogue was 20 000
// of the 79 000 cycles of a 128 x 128 tile with a reduction of 1000.
template <class Core> struct NsTile {
    static constexpr int B = Core::BM, ROW = B * 4, CH = ROW / 16, RPI = 1024 / ROW, INSTR = B * ROW / 1024 / Core::NW;
    static_assert(Core::BM == Core::BN && B * ROW <= Core::LDS, "the tile fits");
    typedef NsQuads<Core> Quads;
    // Where the accumulator quads of a thread lie: rows j of the transposed tile (four consecutive columns i), or, after swap4, row i + t of the tile itself
    // (four consecutive columns).  The wave's, the lane's and the quad's share of a chunk number have no bit in common, so the XOR is one
    // instruction a quad; the low part is four chunks on, which is address bit 6.
    struct Where {
        unsigned t0, tx, u0, ux;                       // row start and chunk swap of either
        __device__ __forceinline__ Where()
        {
            const int lane = threadIdx.x & 63, wave = Core::KW > 1 ? 0 : threadIdx.x >> 6, half = lane >> 5, l = lane & 31, t = l & 3;
            const int wi = (wave / Core::WGN) * (B / Core::WGM), wj = (wave % Core::WGN) * (B / Core::WGN);
            t0 = (wj + l) * ROW + half * 8;
            tx = ((wi / 32 * 8) ^ (l & (CH - 1))) * 16;
            u0 = (wi + half * 4 + t) * ROW + (l & 4) * 2;
            ux = ((wj / 32 * 8 + (l >> 3)) ^ (half * 4 + t)) * 16;
        }
        __device__ __forceinline__ unsigned tile_t(int b) const          // quad b of tile (ti, tj), group g
        {
            const int ti = b / (4 * Core::TN), tj = b / 4 % Core::TN, g = Quads::group(b);
            return t0 + tj * 32 * ROW + (tx ^ ((ti * 8 + g) * 16));
        }
        __device__ __forceinline__ unsigned tile(int b) const
        {
            const int ti = b / (4 * Core::TN), tj = b / 4 % Core::TN, g = Quads::group(b);
            return u0 + (ti * 32 + g * 8) * ROW + (ux ^ (((tj * 8) ^ ((g * 8) & (CH - 1))) * 16));
        }
    };
    static_assert((Core::TN & (Core::TN - 1)) == 0 && (Core::TM & (Core::TM - 1)) == 0, "chunk numbers add without a carry");
    // acc <- alpha acc + beta E;  e: the tile of E^T, `rows` of its rows and `cols` of its columns (a multiple of 32) exist.  Ends with LDS in use.
    static __device__ __forceinline__ void blend(f32x16 (&acc)[Core::TM][Core::TN], float alpha, float beta, const char* e, long ld, int rows, int cols, unsigned char* smem)
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int last = cols >= B ? CH - 1 : cols / 4 - 1;
        e = nt_uniform(e);
        nt_wait_barrier<0>();                                              // everybody is done with what LDS held
#pragma unroll
        for (int q = 0; q < INSTR; ++q) {
            const int k = q * Core::NW + wave, row = k * RPI + lane / CH, c = (lane % CH) ^ (row & (CH - 1));
            nt_dma16(e, (unsigned)((row < rows ? row : rows - 1) * ld + (c < last ? c : last) * 16), (unsigned)(uintptr_t)smem + k * 1024);
        }
        nt_wait_barrier<0>();
        const Where w;
        Quads::each([&](int b, int, int) {
            const unsigned o = w.tile_t(b);
            const f16x4_t h = *(const f16x4_t*)(smem + o), l = *(const f16x4_t*)(smem + (o ^ 64));
            f32x16& c = acc[b / (4 * Core::TN)][b / 4 % Core::TN];
#pragma unroll
            for (int r = 0; r < 4; ++r) c[(b & 3) * 4 + r] = fmaf(alpha, c[(b & 3) * 4 + r], beta * ((float)h[r] + (float)l[r]));
        });
    }
    static __device__ __forceinline__ void copy_out(char* d, long ld, int rows, int cols, unsigned char* smem)
    {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < B * CH / Core::NT; ++k) {
            const int id = k * Core::NT + threadIdx.x, row = id / CH, c = id % CH;
            if (row < rows && (c >> 3) * 32 < cols) *(u32x4*)(d + row * ld + c * 16) = *(const u32x4*)(smem + row * ROW + (c ^ (row & (CH - 1))) * 16);
        }
    }
    // four lanes (columns j & ~3 ..) transpose their 4 x 4 elements: lane t gets row t, four consecutive columns
    static __device__ __forceinline__ u32x2 swap4(u32x2 v)
    {
        const bool s = threadIdx.x & 1, t = threadIdx.x & 2;
        const unsigned p0 = __builtin_amdgcn_update_dpp(0, v[0], 0xB1, 0xf, 0xf, true), p1 = __builtin_amdgcn_update_dpp(0, v[1], 0xB1, 0xf, 0xf, true);
        const unsigned e0 = s ? __builtin_amdgcn_perm(v[0], p0, 0x07060302u) : __builtin_amdgcn_perm(p0, v[0], 0x05040100u);
        const unsigned e1 = s ? __builtin_amdgcn_perm(v[1], p1, 0x07060302u) : __builtin_amdgcn_perm(p1, v[1], 0x05040100u);
        const unsigned y = __builtin_amdgcn_update_dpp(0, t ? e0 : e1, 0x4E, 0xf, 0xf, true);
        return t ? u32x2{y, e1} : u32x2{e0, y};
    }
    // the tile transposed, rows j of the accumulators' columns, to dt; diag: a symmetric tile on the diagonal, see ns_both_halves
    static __device__ __forceinline__ void store_t(const f32x16 (&acc)[Core::TM][Core::TN], float alpha, char* dt, long ld, int rows, int cols, bool diag, unsigned char* smem)
    {
        nt_wait_barrier<0>();
        const Where w;
        Quads::each([&](int b, int i, int j) {
            float q[4];
            Quads::quad(acc, b, q);
#pragma unroll
            for (int r = 0; r < 4; ++r) q[r] *= alpha;
            f16x4_t h, l;
            ns_split4(q, h, l);
            const unsigned o = w.tile_t(b);
            if (!diag) { *(f16x4_t*)(smem + o) = h; *(f16x4_t*)(smem + (o ^ 64)) = l; return; }
            // the lower part twice, mirrored and in its own place; of a 4 x 4 block on the diagonal the row's part up to it, the mirrored part behind it
            const int t = j & 3, j0 = j & ~3;
            if (i < j0) return;                                            // (the four lanes of a swap agree)
            const f16x4_t uh = __builtin_bit_cast(f16x4_t, swap4(__builtin_bit_cast(u32x2, h))), ul = __builtin_bit_cast(f16x4_t, swap4(__builtin_bit_cast(u32x2, l)));
            const unsigned u = w.tile(b);
            if (i == j0) {
#pragma unroll
                for (int r = 0; r < 4; ++r) { h[r] = r <= t ? uh[r] : h[r]; l[r] = r <= t ? ul[r] : l[r]; }
                *(f16x4_t*)(smem + o) = h; *(f16x4_t*)(smem + (o ^ 64)) = l;
            } else {
                *(f16x4_t*)(smem + o) = h; *(f16x4_t*)(smem + (o ^ 64)) = l;
                *(f16x4_t*)(smem + u) = uh; *(f16x4_t*)(smem + (u ^ 64)) = ul;
            }
        });
        copy_out(dt, ld, rows, cols, smem);
    }
    // the tile itself to d
    static __device__ __forceinline__ void store(const f32x16 (&acc)[Core::TM][Core::TN], float alpha, char* d, long ld, int rows, int cols, unsigned char* smem)
    {
        nt_wait_barrier<0>();
        const Where w;
        Quads::each([&](int b, int, int) {
            float q[4];
            Quads::quad(acc, b, q);
#pragma unroll
            for (int r = 0; r < 4; ++r) q[r] *= alpha;
            f16x4_t h, l;
            ns_split4(q, h, l);
            const unsigned u = w.tile(b);
            *(u32x2*)(smem + u) = swap4(__builtin_bit_cast(u32x2, h));
            *(u32x2*)(smem + (u ^ 64)) = swap4(__builtin_bit_cast(u32x2, l));
        });
        copy_out(d, ld, rows, cols, smem);
    }
};

// tile t of the lower triangle of nt x nt tiles: (ti, tj), tj <= ti.  Walked in blocks of 8 x 8 tiles, so that the tiles in flight on one XCD share
// eight row panels of either operand.
__device__ __forceinline__ int ns_row(int t)          // row of t in a triangle walked row by row
{
    int i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    return i;
}
__device__ __forceinline__ void ns_lower(int t, int nt, int& ti, int& tj)
{
    int I = (int)((sqrtf(16.f + 128.f * (float)t) - 4.f) * (1.f / 64.f));         // block rows before I hold 32 I^2 + 4 I tiles
    while (32 * (I + 1) * (I + 1) + 4 * (I + 1) <= t) ++I;
    while (32 * I * I + 4 * I > t) --I;
    t -= 32 * I * I + 4 * I;
    const int h = nt - 8 * I < 8 ? nt - 8 * I : 8;
    if (t < h * 8 * I) { ti = 8 * I + t % h; tj = t / h; return; }
    t -= h * 8 * I;
    const int r = ns_row(t);
    ti = 8 * I + r; tj = 8 * I + t - r * (r + 1) / 2;
}

// Workgroup ids go round the eight XCDs, each with an L2 of its own.  XCD x takes the x-th of eight runs of equal cost of the list, so that the tiles of a
// matrix meet in one L2: dealt out one by one, six 1000 x 1024 matrices were read into all eight (220 MB a launch, 45 us at the rate of the fabric).
struct NsDeal { int b[9]; };
__device__ __forceinline__ int ns_dealt(const NsDeal& d, int id)
{
    const int x = id & 7, t = d.b[x] + (id >> 3);
    return t < d.b[x + 1] ? t : -1;
}

// D = alpha A B^T (+ beta E + gamma F + diag I) for a symmetric D -- X X^T, or a product of symmetric matrices that commute: lower tiles, both halves
// written.  blockIdx.y picks the product: the two of one phase are independent.  The tiles behind the first split.full are cut along the reduction into
// split.s parts, whose float32 sums go to memory in accumulator order for ns_finish_kernel.
struct NsProd { int a, b, e, f, d; float alpha, beta, gamma, diag; };          // diag: added to the diagonal of a product with an E
struct NsProds {
    NsProd p[2];
    __device__ __forceinline__ NsProd of(int y) const
    {
        const NsProd u = p[0], v = p[1];
        return NsProd{y ? v.a : u.a, y ? v.b : u.b, y ? v.e : u.e, y ? v.f : u.f, y ? v.d : u.d, y ? v.alpha : u.alpha, y ? v.beta : u.beta, y ? v.gamma : u.gamma, y ? v.diag : u.diag};
    }
};

// The waves of a shared reduction add their sums, in the order of the waves: wave w ends with quad w of each lane
template <class Core> __device__ __forceinline__ void ns_join(f32x16 (&acc)[Core::TM][Core::TN], unsigned char* smem)
{
    static_assert(Core::KW == 4 && Core::NW == 4 && Core::LDS >= 16384, "a 32 x 32 tile");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    nt_wait_barrier<0>();
    f32x4* s = (f32x4*)smem;
#pragma unroll
    for (int g = 0; g < 4; ++g) s[(wave * 4 + g) * 64 + lane] = f32x4{acc[0][0][g * 4], acc[0][0][g * 4 + 1], acc[0][0][g * 4 + 2], acc[0][0][g * 4 + 3]};
    __syncthreads();
    f32x4 c = s[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) { const f32x4 x = s[(w * 4 + wave) * 64 + lane]; for (int r = 0; r < 4; ++r) c[r] += x[r]; }
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[0][0][r] = c[r];
}

// blends E and F into a whole tile and stores it with its mirror image
template <class Core> __device__ __forceinline__ void ns_prod_end(const NsView& v, const NsProd& p, float alpha, int ti, int tj, f32x16 (&acc)[Core::TM][Core::TN], unsigned char* smem)
{
    typedef NsTile<Core> Tile;
    constexpr int T = Core::BM;
    const long ls = (long)v.mp * 4, oij = (long)ti * T * ls + tj * T * 4, oji = (long)tj * T * ls + ti * T * 4;       // tile (ti, tj) and its mirror image
    const int ri = v.mp - ti * T, rj = v.mp - tj * T;
    if (p.e >= 0) { Tile::blend(acc, alpha, p.beta, v.sym(p.e) + oji, ls, rj, ri, smem); alpha = 1.f; }
    if (p.f >= 0) Tile::blend(acc, alpha, p.gamma, v.sym(p.f) + oji, ls, rj, ri, smem);
    if (p.diag != 0.f && ti == tj)
        NsQuads<Core>::each([&](int b, int i, int j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[b / (4 * Core::TN)][b / 4 % Core::TN][(b & 3) * 4 + r] += i + r == j ? p.diag : 0.f;
        });
    Tile::store_t(acc, alpha, v.sym(p.d) + oji, ls, rj, ri, ti == tj, smem);
    if (ti != tj) Tile::store(acc, alpha, v.sym(p.d) + oij, ls, ri, rj, smem);
}
template <class Core> __global__ __launch_bounds__(Core::NT, 512 / Core::NT) void ns_prod_kernel(NsTable tab, int kind, NsProds pr, float grown, NsDeal deal, int tail)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    constexpr int T = Core::BM;
    // (deal ends at the first cut tile of a single matrix: its parts follow in launch order, behind a whole number of rounds)
    const int id = (int)blockIdx.x < tail ? ns_dealt(deal, blockIdx.x) : deal.b[8] + (int)blockIdx.x - tail;
    if (id < 0) return;
    const NsProd p = pr.of(blockIdx.y);
    const NsItem it = ns_item(tab, id, [&](const NsItem& t) { return t.split[kind].p; });
    const NsView v(it);
    const NsSplit sl = it.of(kind);
    const int nt = (v.mp + T - 1) / T, cut = nt * (nt + 1) / 2 - sl.full;
    int t = id - sl.p, sp = 0, parts = 1, ti, tj;
    if (t >= sl.full) { sp = (t - sl.full) / cut; t = sl.full + (t - sl.full) % cut; parts = sl.s; }       // neighbours work on one stretch of the reduction
    ns_lower(t, nt, ti, tj);
    const int steps = (p.a == NS_X ? v.np : v.mp) * 4 / Core::RB, k0 = (int)((long)steps * sp / parts), k1 = (int)((long)steps * (sp + 1) / parts);
    const long ld = (long)steps * Core::RB;
    const char* a = (p.a == NS_X ? v.x : v.sym(p.a)) + (long)k0 * Core::RB;
    const char* b = (p.a == NS_X ? v.x : v.sym(p.b)) + (long)k0 * Core::RB;
    const float t2 = p.a == NS_X ? v.t(grown) * v.t(grown) : 1.f;
    f32x16 acc[Core::TM][Core::TN] = {};
    Core::run(a + ti * T * ld, (unsigned)ld, v.mp - ti * T, b + tj * T * ld, (unsigned)ld, v.mp - tj * T, k1 - k0, smem, acc);
    if constexpr (Core::KW > 1) ns_join<Core>(acc, smem);
    typedef NsQuads<Core> Quads;
    if (parts > 1) {
        float* d = v.part() + (((long)blockIdx.y * cut + t - sl.full) * parts + sp) * Quads::FLOATS + threadIdx.x * 4;
        Quads::each([&](int b, int, int) { float q[4]; Quads::quad(acc, b, q); *(f32x4*)(d + b * Core::NT * 4) = f32x4{q[0], q[1], q[2], q[3]}; });
        return;
    }
    ns_prod_end<Core>(v, p, p.alpha * t2, ti, tj, acc, smem);
}
// one accumulator quad of a cut tile a thread; blockIdx.x = tile * quads + quad
template <class Core> __global__ __launch_bounds__(Core::NT) void ns_finish_kernel(NsTable tab, int kind, NsProds pr, float grown)
{
    constexpr int T = Core::BM, N = NsQuads<Core>::N;
    const int id = blockIdx.x / N, q = blockIdx.x % N;
    const NsProd p = pr.of(blockIdx.y);
    const NsItem it = ns_item(tab, id, [&](const NsItem& t) { return t.split[kind].c; });
    const NsSplit sl = it.of(kind);
    const int t = sl.full + id - sl.c;
    const NsView v(it);
    const int nt = (v.mp + T - 1) / T, cut = nt * (nt + 1) / 2 - sl.full;
    int ti, tj, i, j;
    ns_lower(t, nt, ti, tj);
    NsQuads<Core>::at(q, i, j);
    const float* s = v.part() + (((long)blockIdx.y * cut + t - sl.full) * sl.s) * NsQuads<Core>::FLOATS + q * Core::NT * 4 + threadIdx.x * 4;
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int sp = 0; sp < sl.s; ++sp) { const f32x4 w = *(const f32x4*)(s + (long)sp * NsQuads<Core>::FLOATS); for (int r = 0; r < 4; ++r) c[r] += w[r]; }
    i += ti * T; j += tj * T;
    if (i >= v.mp || j >= v.mp) return;
    const long ls = (long)v.mp * 4;
    const float alpha = p.a == NS_X ? p.alpha * (v.t(grown) * v.t(grown)) : p.alpha;
    float w[4], x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) w[r] = alpha * c[r];
    if (p.e >= 0) {
        ns_read4(v.sym(p.e), ls, j, i, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fmaf(p.beta, x[r], w[r]);
    }
    if (p.f >= 0) {
        ns_read4(v.sym(p.f), ls, j, i, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fmaf(p.gamma, x[r], w[r]);
    }
    char* d = v.sym(p.d);
    if (ti == tj) {
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] += i + r == j ? p.diag : 0.f;
        ns_both_halves(i, j, w, [&](int r, int c, const Pair& e) { char* o = d + r * ls + (c >> 5) * 128 + (c & 31) * 2; *(_Float16*)o = e.h; *(_Float16*)(o + 64) = e.l; });
        return;
    }
    f16x4_t h, l;
    ns_split4(w, h, l);
    char* o = d + j * ls + (i >> 5) * 128 + (i & 31) * 2;
    *(f16x4_t*)o = h; *(f16x4_t*)(o + 64) = l;
#pragma unroll
    for (int r = 0; r < 4; ++r) { char* m = d + (i + r) * ls + (j >> 5) * 128 + (j & 31) * 2; *(_Float16*)m = h[r]; *(_Float16*)(m + 64) = l[r]; }
}

__device__ __forceinline__ void ns_rates(const float* hyper, int rows, int cols, int adjust, float& keep, float& rate)
{
    const float lr = hyper[0];
    keep = 1.f - lr * hyper[2];
    rate = lr * (adjust ? 0.2f * sqrtf((float)(rows > cols ? rows : cols)) : rows > cols ? sqrtf((float)rows / (float)cols) : 1.f);
}

// X <- alpha Q X + beta X.  MODE 0: back to X and the other X^T; 1: to the caller's matrix; 2: the Muon update of the caller's parameter
template <class Core, typename T, int MODE> __global__ __launch_bounds__(Core::NT, 512 / Core::NT) void ns_apply_kernel(NsTable tab, int q, int xt, float alpha, float beta, float grown, float grown_to, const float* __restrict__ hyper, int adjust, NsDeal deal)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    constexpr int B = Core::BM;
    const int id = ns_dealt(deal, blockIdx.x);
    if (id < 0) return;
    const NsItem it = ns_item(tab, id, [&](const NsItem& t) { return t.p_app; });
    const NsView v(it);
    int ti, tj;
    nt_band(id - it.p_app, (v.np + B - 1) / B, (v.mp + B - 1) / B, tj, ti);
    const float t = MODE == 0 ? v.t(grown) / v.t(grown_to) : v.t(grown);          // (powers of two)
    alpha *= t; beta *= t;
    f32x16 acc[Core::TM][Core::TN] = {};
    const long ld = (long)v.mp * 4;
    Core::run(v.sym(q) + ti * B * ld, (unsigned)ld, v.mp - ti * B, v.xt(xt) + tj * B * ld, (unsigned)ld, v.np - tj * B, v.mp * 4 / Core::RB, smem, acc);
    if constexpr (Core::KW > 1) ns_join<Core>(acc, smem);
    typedef NsQuads<Core> Quads;
    typedef NsTile<Core> Tile;
    const long oji = (long)tj * B * ld + ti * B * 4;
    const int ri = v.mp - ti * B, rj = v.np - tj * B;
    Tile::blend(acc, alpha, beta, v.xt(xt) + oji, ld, rj, ri, smem);
    if (MODE == 0) {
        Tile::store_t(acc, 1.f, v.xt(xt ^ 1) + oji, ld, rj, ri, false, smem);
        Tile::store(acc, 1.f, v.x + (long)ti * B * v.np * 4 + tj * B * 4, v.np * 4L, ri, rj, smem);
        return;
    }
    const long si = v.tall ? 1 : it.ld_dst, sj = v.tall ? it.ld_dst : 1;
    T* d = (T*)it.dst + ti * B * si + tj * B * sj;
    const int mi = v.m - ti * B, nj = v.n - tj * B;
    if (MODE == 2) {
        float keep, rate, old[Quads::N][4];
        ns_rates(hyper, it.rows, it.cols, adjust, keep, rate);
        Quads::each([&](int b, int i, int j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) old[b][r] = i + r < mi && j < nj ? (float)d[(i + r) * si + j * sj] : 0.f;
        });
        Quads::each([&](int b, int i, int j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) if (i + r < mi && j < nj) d[(i + r) * si + j * sj] = (T)fmaf(-rate, acc[b / (4 * Core::TN)][b / 4 % Core::TN][(b & 3) * 4 + r], keep * old[b][r]);
        });
        return;
    }
    Quads::each([&](int b, int i, int j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) if (i + r < mi && j < nj) ns_store(d + (i + r) * si + j * sj, acc[b / (4 * Core::TN)][b / 4 % Core::TN][(b & 3) * 4 + r]);
    });
}

// ---- short matrices: up to 32 rows (or columns), three launches -----------------------------------------------------------------------------
// The iteration is W(S) X0 with one polynomial W of S = X0 X0^T.  With 32 rows S is so small that it can be kept in FLOAT64, where composing ALL steps is
// sound (an error grows by a^2 = 12 a step from 2^-53): one pass over the matrix for S, whose trace is the norm, one workgroup for W, one pass
// for W X0.  The float64 rate of the vector units equals the float32 one, and both passes move little else than the matrix.
constexpr int NSS_COLS = 64;                   // columns of the long side a workgroup stages at once
struct NssItem { const void* src; void* dst; float* buf; int ld_src, ld_dst, rows, cols, p, tiles; };       // tiles: of NSS_COLS, a workgroup
constexpr int NSS_CHUNK = 80;
struct NssItems { double* ws; NssItem it[NSS_CHUNK]; };       // ws: 1024 numbers for every workgroup and for every matrix
__device__ __forceinline__ double* nss_ws(const NssItems& items, int i) { return items.ws + (long)(items.it[i].p + i) * 1024; }
static_assert(sizeof(NssItems) <= 4032, "kernel arguments end at 4 KB");

// columns c0 .. c0 + 63 of the matrix (long side) into s[32][68], zeros outside
template <typename T, bool MUON, bool STORE> __device__ __forceinline__ void nss_stage(const NssItem& it, int c0, const float* __restrict__ hyper, float (*s)[68])
{
    const bool tall = it.rows > it.cols;
    const int m = tall ? it.cols : it.rows, n = tall ? it.rows : it.cols;
    float h[5] = {0.f, 0.f, 0.f, 0.f, 1.f};
    if (MUON) for (int i = 0; i < 5; ++i) h[i] = hyper[i];
#pragma unroll
    for (int q = 0; q < 32 * NSS_COLS / 256; ++q) {
        const int k = threadIdx.x + q * 256, i = tall ? k & 31 : k >> 6, c = tall ? k >> 5 : k & 63, j = c0 + c;
        float u = 0.f;
        if (i < m && j < n) {
            const long r = tall ? j : i, e = tall ? i : j;
            u = ns_load((const T*)it.src + r * it.ld_src + e);
            if (MUON) {
                float* b = it.buf + r * it.cols + e;
                float o = *b;
                if (STORE) { o = ns_momentum(u, o, h); *b = o; }
                u = ns_update(u, o, h);
            }
        }
        s[i][c] = u;
    }
}
template <typename T, bool MUON> __global__ __launch_bounds__(256) void nss_gram_kernel(NssItems items, int count, const float* __restrict__ hyper)
{
    __shared__ __attribute__((aligned(16))) float s_x[32][68];
    __shared__ double s_g[4][32][33];
    const int id = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, a0 = (tid >> 3 & 7) * 4, b0 = (tid & 7) * 4;
    const int which = ns_find(count, id, [&](int i) { return items.it[i].p; });
    const NssItem it = items.it[which];
    double acc[4][4] = {};
    const int n = it.rows > it.cols ? it.rows : it.cols, first = (id - it.p) * it.tiles;
    for (int t = 0; t < it.tiles && (first + t) * NSS_COLS < n; ++t) {
        if (t) __syncthreads();
        nss_stage<T, MUON, true>(it, (first + t) * NSS_COLS, hyper, s_x);
        __syncthreads();
        // a wave: 16 of the columns, a thread 4 x 4 of the sums
#pragma unroll 2
        for (int k = wave * 16; k < wave * 16 + 16; k += 4) {
            f32x4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = *(const f32x4*)&s_x[a0 + i][k]; b[i] = *(const f32x4*)&s_x[b0 + i][k]; }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fma((double)a[i][e], (double)b[j][e], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_g[wave][a0 + i][b0 + j] = acc[i][j];
    __syncthreads();
    double* g = nss_ws(items, which) + (long)(1 + id - it.p) * 1024;
    for (int k = tid; k < 1024; k += 256) g[k] = (s_g[0][k >> 5][k & 31] + s_g[1][k >> 5][k & 31]) + (s_g[2][k >> 5][k & 31] + s_g[3][k >> 5][k & 31]);
}

typedef __attribute__((ext_vector_type(4))) double f64x4;
typedef __attribute__((ext_vector_type(2))) double f64x2;
typedef double NssMat[32][34];          // rows 16 bytes apart in the banks: the 16-byte reads of 16 rows meet in none
// quadrant `quad` of A B for symmetric A, B: element r of lane l is (row l / 16 + 4 r, column l % 16) of it.  A lane group takes eight neighbouring indices of
// the sum, two a read; two chains, because the MFMAs of one wait for each other.
__device__ __forceinline__ f64x4 nss_product(const NssMat& a, const NssMat& b, int quad)
{
    const int lane = threadIdx.x & 63, i = (quad >> 1) * 16 + (lane & 15), j = (quad & 1) * 16 + (lane & 15), k = (lane >> 4) * 8;
    f64x2 x[4], y[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) { x[s] = *(const f64x2*)&a[i][k + 2 * s]; y[s] = *(const f64x2*)&b[j][k + 2 * s]; }
    f64x4 c = {0.0, 0.0, 0.0, 0.0}, d = c;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[s][0], y[s][0], c, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(x[s][1], y[s][1], d, 0, 0, 0);
    }
    return c + d;
}
// W / norm from the sums of nss_gram_kernel: a workgroup a matrix, waves 0 - 3 and 4 - 7 a product each.  S' = (a I + P)^2 S, W' = (a I + P) W.
__global__ __launch_bounds__(512) void nss_poly_kernel(NssItems items, int steps, double a, double b, double c, float eps)
{
    __shared__ __attribute__((aligned(16))) NssMat S, P, R, W;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = wave & 3;
    const NssItem it = items.it[blockIdx.x];
    double* ws = nss_ws(items, blockIdx.x);
    const int n = it.rows > it.cols ? it.rows : it.cols, parts = (n + it.tiles * NSS_COLS - 1) / (it.tiles * NSS_COLS);
    for (int k = tid; k < 1024; k += 512) {
        double sum = 0.0;
#pragma unroll 8
        for (int p = 0; p < parts; ++p) sum += ws[(long)(1 + p) * 1024 + k];
        S[k >> 5][k & 31] = sum;
    }
    __syncthreads();
    double trace = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) trace += S[i][i];
    double norm = sqrt(trace);
    if (norm <= (double)eps) norm = (double)eps;                          // a NaN norm stays NaN
    const double inv = 1.0 / (norm * norm);
    __syncthreads();
    for (int k = tid; k < 1024; k += 512) { S[k >> 5][k & 31] *= inv; W[k >> 5][k & 31] = (k >> 5) == (k & 31) ? 1.0 / norm : 0.0; }
    __syncthreads();
    const int j = (quad & 1) * 16 + (lane & 15), i0 = (quad >> 1) * 16 + (lane >> 4);
    for (int st = 0; st < steps; ++st) {
        f64x4 x = {0.0, 0.0, 0.0, 0.0};
        if (wave < 4) {
            x = nss_product(S, S, quad);
#pragma unroll
            for (int r = 0; r < 4; ++r) P[i0 + 4 * r][j] = b * S[i0 + 4 * r][j] + c * x[r] + (i0 + 4 * r == j ? a : 0.0);      // a I + b S + c S^2
        }
        __syncthreads();
        x = wave < 4 ? nss_product(P, S, quad) : nss_product(P, W, quad);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) (wave < 4 ? R : W)[i0 + 4 * r][j] = x[r];
        __syncthreads();
        if (wave < 4 && st + 1 < steps) {
            x = nss_product(R, P, quad);
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i0 + 4 * r][j] = x[r];
        }
        __syncthreads();
    }
    for (int k = tid; k < 1024; k += 512) ws[k] = W[k >> 5][k & 31];
}
template <typename T, bool MUON> __global__ __launch_bounds__(256) void nss_apply_kernel(NssItems items, int count, const float* __restrict__ hyper, int adjust)
{
    __shared__ __attribute__((aligned(16))) float s_x[32][68];
    __shared__ __attribute__((aligned(16))) double s_w[32][34];
    const int id = blockIdx.x, tid = threadIdx.x;
    const int which = ns_find(count, id, [&](int i) { return items.it[i].p; });
    const NssItem it = items.it[which];
    for (int k = tid; k < 1024; k += 256) s_w[k >> 5][k & 31] = nss_ws(items, which)[k];
    const bool tall = it.rows > it.cols;
    const int m = tall ? it.cols : it.rows, n = tall ? it.rows : it.cols, first = (id - it.p) * it.tiles;
    float keep = 0.f, rate = 0.f;
    if (MUON) ns_rates(hyper, it.rows, it.cols, adjust, keep, rate);
    // a thread: 2 rows x 4 columns; lanes run along the caller's contiguous side
    const int i0 = (tall ? tid & 15 : tid >> 4) * 2, c0 = (tall ? tid >> 4 : tid & 15) * 4;
    for (int t = 0; t < it.tiles && (first + t) * NSS_COLS < n; ++t) {
        __syncthreads();
        const int base = (first + t) * NSS_COLS;
        nss_stage<T, MUON, false>(it, base, hyper, s_x);
        __syncthreads();
        T old[2][4];
        auto at = [&](int i, int j) { return (T*)it.dst + (tall ? (long)(base + c0 + j) * it.ld_dst + i0 + i : (long)(i0 + i) * it.ld_dst + base + c0 + j); };
        if (MUON)                                                          // on its way while the sums are formed
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) old[i][j] = i0 + i < m && base + c0 + j < n ? *at(i, j) : T(0);
        double acc[2][4] = {};
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
            const f32x4 x = *(const f32x4*)&s_x[k][c0];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const double w = s_w[k][i0 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fma(w, (double)x[j], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i0 + i >= m || base + c0 + j >= n) continue;
                if (MUON) *at(i, j) = (T)fmaf(-rate, (float)acc[i][j], keep * (float)old[i][j]);
                else ns_store(at(i, j), (float)acc[i][j]);
            }
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------------------------------
static int ns_check(const saunet_ns_desc* d, const char* who)
{
    if (!d || !d->item || d->count < 1 || d->count > 4096) return set_error(SAUNET_BAD_SHAPE, "%s: 1 to 4096 matrices, not %d", who, d ? d->count : 0);
    if (d->dtype != SAUNET_F32 && d->dtype != SAUNET_BF16 && d->dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "%s: dtype %d", who, d->dtype);
    if (d->steps < 1 || d->steps > 32) return set_error(SAUNET_BAD_SHAPE, "%s: 1 to 32 steps, not %d", who, d->steps);
    if (!(d->eps > 0.f) || !(fabsf(d->a) <= 4096.f) || !(fabsf(d->b) <= 4096.f) || !(fabsf(d->c) <= 4096.f)) return set_error(SAUNET_BAD_SHAPE, "%s: eps has to be positive, the coefficients finite and below 4096", who);
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        if (t.rows < 1 || t.cols < 1 || t.rows > (1 << 20) || t.cols > (1 << 20) || (t.rows > 32768 && t.cols > 32768))
            return set_error(SAUNET_BAD_SHAPE, "%s: matrix %d is %d x %d (sides up to 2^20, the shorter up to 32768)", who, i, t.rows, t.cols);
        if (t.ld_src < t.cols || t.ld_dst < t.cols || t.ld_src > 0x7fffffff || t.ld_dst > 0x7fffffff) return set_error(SAUNET_BAD_SHAPE, "%s: matrix %d has a bad row stride", who, i);
    }
    return SAUNET_OK;
}

// One call: the matrices with up to 32 rows go one way, the others the other way
struct NsPlan { long small, large, small_at, norm, pack, tile, app, grid[NS_KINDS], cut[NS_KINDS], tab_at, part_at, bytes, shortest; int tile_g, tile_m, tile_n; NsDeal deal[NS_KINDS + 1]; };

static bool ns_is_small(const saunet_ns_desc* d, const saunet_ns_item& t)
{
    // all steps composed in float64: 2^-53 a^(2 (steps - 1)) has to stay below float32's rounding
    double grow = 1.0;
    for (int i = 1; i < d->steps; ++i) grow *= (double)d->a * d->a;
    return (t.rows < t.cols ? t.rows : t.cols) <= 32 && grow <= 1e8;
}
// Cuts along the reduction, for one kind of launch (ny products a tile, steps[i] reduction steps of matrix i; none if `whole`).  A tile longer than an even share of the
// launch's work is cut into shares (sixteen steps at least) where that saves 32 steps: they are 11 us, the finishing launch costs 8 (six 1000 x 1024
// matrices in two parts of sixteen: 41 -> 33 us for the products, 14 more to finish).  A single matrix of a few rounds of NS_SLOTS workgroups whose last
// round is less than half full has that round's tiles cut: 4096 x 4096, 528 tiles on 512 slots, 262 us -> 200 + 11.
static void ns_cut(int kind, int ny, bool whole, NsPlan& p, const int* tiles, const int* steps, int count, NsItem* out)
{
    long total = 0, at = 0, work = 0;
    for (int i = 0; i < count; ++i) { total += (long)tiles[i] * ny; work += (long)tiles[i] * ny * steps[i]; }
    const long share = work / NS_SLOTS > 16 ? work / NS_SLOTS : 16;
    long tail = 0, tail_s = 1;
    if (!whole && count == 1 && total > NS_SLOTS && total < 4 * NS_SLOTS && total % NS_SLOTS && total % NS_SLOTS <= NS_SLOTS / 2) {
        tail = (total % NS_SLOTS + ny - 1) / ny;
        tail_s = NS_SLOTS / (tail * ny);
        if (tail_s > steps[0] / 8) tail_s = steps[0] / 8;
        if (tail_s < 2) { tail = 0; tail_s = 1; }
    }
    p.cut[kind] = 0;
    for (int i = 0; i < count; ++i) {
        NsSplit s = {(int)at, tiles[i], 1, (int)p.cut[kind]};
        if (tail) { s.full = tiles[i] - (int)tail; s.s = (int)tail_s; }
        else if (!whole && steps[i] >= share + 32) { s.full = 0; s.s = (int)((steps[i] + share - 1) / share); }
        p.cut[kind] += tiles[i] - s.full;
        at += s.full + (long)(tiles[i] - s.full) * s.s;
        out[i].split[kind] = s;
    }
    p.grid[kind] = at;
}

// Runs of equal cost for the XCDs: runs[r] = {workgroups, cost of one}, in launch order
struct NsRun { long n; long cost; };
constexpr int NS_FIXED = 8;                  // start and end of a tile, in reduction steps
static NsDeal ns_deal(const NsRun* run, int runs)
{
    NsDeal d = {};
    long total = 0, before = 0, at = 0;
    for (int r = 0; r < runs; ++r) total += run[r].n * run[r].cost;
    int x = 1;
    for (int r = 0; r < runs; ++r) {
        for (; x < 8; ++x) {
            const long need = total * x / 8 - before;                     // border x falls into this run?
            if (need > run[r].n * run[r].cost) break;
            d.b[x] = (int)(at + (need + run[r].cost / 2) / run[r].cost);
        }
        before += run[r].n * run[r].cost; at += run[r].n;
    }
    for (; x < 9; ++x) d.b[x] = (int)at;
    d.b[8] = (int)at;
    return d;
}
static unsigned ns_deal_grid(const NsDeal& d)
{
    int most = 0;
    for (int x = 0; x < 8; ++x) if (d.b[x + 1] - d.b[x] > most) most = d.b[x + 1] - d.b[x];
    return 8u * most;
}

// `large` and `small`: the items of either way (capacity 4096), laid out against workspace `ws`.  Workspace: table | norm partials | matrices
static int ns_plan(const saunet_ns_desc* d, NsPlan& p, NsItem* large, NssItem* small, char* ws)
{
    static thread_local int tiles[2][4096], gram[4096], sym[4096];
    p = NsPlan();
    long a128 = 0, g128 = 0, w64 = 0, a64 = 0, longest = 0;
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        const long m = t.rows < t.cols ? t.rows : t.cols, n = t.rows < t.cols ? t.cols : t.rows;
        if (ns_is_small(d, t)) {
            NssItem& o = small[p.small++];
            o.src = t.src; o.dst = t.dst; o.buf = (float*)t.buf; o.ld_src = (int)t.ld_src; o.ld_dst = (int)t.ld_dst; o.rows = t.rows; o.cols = t.cols;
            const long cols = (n + NSS_COLS - 1) / NSS_COLS;
            o.tiles = (int)((cols + 63) / 64);                  // 64 workgroups a matrix at most: their sums are added by one
            o.p = (int)((cols + o.tiles - 1) / o.tiles);        // (a count for now)
            continue;
        }
        NsItem& o = large[p.large++];
        o.src = t.src; o.dst = t.dst; o.buf = (float*)t.buf; o.ld_src = (int)t.ld_src; o.ld_dst = (int)t.ld_dst; o.rows = t.rows; o.cols = t.cols;
        a128 += (m + 127) / 128 * ((n + 127) / 128);
        w64 += (m + 63) / 64 * ((m + 63) / 64 + 1) / 2;
        a64 += (m + 63) / 64 * ((n + 63) / 64);
        longest = n > longest ? n : longest;
        g128 += (m + 127) / 128 * ((m + 127) / 128 + 1) / 2 * ((n + 31) / 32);
        if (p.large == 1 || m < p.shortest) p.shortest = m;
    }
    // the longest reductions first: what starts last is short
    std::sort(large, large + p.large, [](const NsItem& x, const NsItem& y) { return (x.rows < x.cols ? x.rows : x.cols) > (y.rows < y.cols ? y.rows : y.cols); });
    // 64 x 64 tiles where 128 x 128 ones would leave CUs idle or be mostly padding (us a call, replayed; 128 against 64).
    // m x m products: as long as the small tiles fill the NS_SLOTS once (1200 x 1300 548 -> 364, 1900 x 2000 865 -> 738, fourteen 500 x 1000 450 -> 391; but
    // fifteen 512 x 512, 540 tiles, 401 -> 425) or what starts behind that is short (the network's 162 matrices, one of 1000 rows and 60 of 128: 1202 -> 1102),
    // and twice where the reductions are long (2200^2, 630, 1268 -> 1179; two 1500^2, 600, 917 -> 863; but four 1000 x 1024, 544, 570 -> 618).
    // Gram products: by their steps (300 x 3000, 564: 150 -> 139; 512 x 4000, 1250: 179 -> 172; but 512 x 8000, 2500: 203 -> 211), and of short sums as the m x m ones
    // (1900 x 2000 738 -> 716, thirteen 512 x 512 334 -> 325; but 1000 x 3000 342 -> 352).
    // Products with X: by their tiles (1000 x 1024, 64: 335 -> 304; 512 x 4000, 128: 188 -> 179; but three 1000 x 1024, 192: 535 -> 542).
    long second = 0, longest_m = 0;                                       // rows of the first small tile of the second round, of the first
    for (long i = 0, at = 0; i < p.large && !second; ++i) {
        const long m = large[i].rows < large[i].cols ? large[i].rows : large[i].cols;
        if (!i) longest_m = m;
        at += (m + 63) / 64 * ((m + 63) / 64 + 1) / 2;
        if (at > NS_SLOTS) second = m;
    }
    p.tile_m = second * 4 <= longest_m || (w64 <= 2 * NS_SLOTS && p.shortest >= 1200) ? 64 : 128;
    p.tile_g = g128 <= 1400 || (p.tile_m == 64 && longest <= 2560) ? 64 : 128;
    p.tile_n = a128 <= 128 ? 64 : 128;
    // 32 x 32 tiles, whose waves share one reduction, where even the 64 x 64 ones leave CUs idle: four times the workgroups, a third of the LDS traffic in each
    // (us a call, replayed; 64 against 32).  m x m products: 3 tiles of 64 98 -> 92, 36 196 -> 156, 90 117 -> 113, but 136 302 -> 337.  Products with X: 8 tiles
    // 92 -> 86, 126 119 -> 115, but 188 142 -> 144, 240 113 -> 125.  Gram products where they would not be cut: 128 x 1000 130 -> 103, 768 x 1000
    // 202 -> 194, but 512 x 2000 156 -> 156, 200 x 3000 142 -> 160.
    if (p.tile_m == 64 && w64 <= 96) p.tile_m = 32;
    if (p.tile_n == 64 && a64 <= 128) p.tile_n = 32;
    if (p.tile_g == 64 && w64 <= 96 && longest < 1536) p.tile_g = 32;
    for (long i = 0; i < p.large; ++i) {
        NsItem& o = large[i];
        const long m = o.rows < o.cols ? o.rows : o.cols, n = o.rows < o.cols ? o.cols : o.rows, mp = (m + 63) / 64 * 64, np = (n + 63) / 64 * 64;
        const long tm = (mp + p.tile_m - 1) / p.tile_m, tg = (mp + p.tile_g - 1) / p.tile_g;
        o.p_norm = (int)p.norm; o.p_pack = (int)p.pack; o.p_app = (int)p.app;
        tiles[0][i] = (int)(tg * (tg + 1) / 2); tiles[1][i] = (int)(tm * (tm + 1) / 2); gram[i] = (int)(np / 32); sym[i] = (int)(mp / 32);
        p.norm += (m * n + NS_NORM - 1) / NS_NORM;
        p.pack += ((mp + 63) / 64) * ((np + 63) / 64);
        p.app += ((mp + p.tile_n - 1) / p.tile_n) * ((np + p.tile_n - 1) / p.tile_n);
        p.tile += tiles[1][i] + tiles[0][i];
        if (p.norm > 0x3fffffff || p.pack > 0x3fffffff || p.app > 0x3fffffff || p.tile > 0x3ffffff) return set_error(SAUNET_BAD_SHAPE, "newton_schulz: the list is too large for one call");
    }
    if (p.large) {
        ns_cut(NS_GRAM, 1, p.tile_g == 32, p, tiles[0], gram, (int)p.large, large);
        ns_cut(NS_ONE, 1, p.tile_m == 32, p, tiles[1], sym, (int)p.large, large);
        ns_cut(NS_TWO, 2, p.tile_m == 32, p, tiles[1], sym, (int)p.large, large);
        static thread_local NsRun run[2 * 4096];
        for (int k = 0; k < NS_KINDS; ++k) {
            int n = 0;
            for (long i = 0; i < p.large; ++i) {
                const NsSplit& sp = large[i].split[k];
                const int steps = k == NS_GRAM ? gram[i] : sym[i], all = tiles[k != NS_GRAM][i];
                if (sp.full) run[n++] = NsRun{sp.full, steps + NS_FIXED};
                if (all > sp.full && !sp.full) run[n++] = NsRun{(long)(all - sp.full) * sp.s, steps / sp.s + NS_FIXED};
            }
            p.deal[k] = ns_deal(run, n);
        }
        for (long i = 0; i < p.large; ++i) run[i] = NsRun{(i + 1 < p.large ? large[i + 1].p_app : p.app) - large[i].p_app, sym[i] + NS_FIXED};
        p.deal[NS_KINDS] = ns_deal(run, (int)p.large);
    }
    long at = 0;
    auto take = [&](long bytes) { const long r = at; at += (bytes + 255) / 256 * 256; return r; };
    p.tab_at = take((long)sizeof(NsItem) * p.large);
    p.part_at = take(p.norm * 8);
    for (long i = 0; i < p.large; ++i) {
        long cut = 0;
        for (int k = 0; k < NS_KINDS; ++k) {
            const NsSplit& s = large[i].split[k];
            const long side = k == NS_GRAM ? p.tile_g : p.tile_m;
            const long c = s.s > 1 ? (long)(tiles[k != NS_GRAM][i] - s.full) * s.s * (k == NS_TWO ? 2 : 1) * side * side * 4 : 0;
            if (c > cut) cut = c;
        }
        large[i].ws = ws + take(NsView::bytes(large[i].rows, large[i].cols) + cut);
    }
    p.small_at = at;
    for (long i = 0; i < p.small; ++i) take((long)(small[i].p + 1) * 1024 * 8);
    p.bytes = at + 256;
    return SAUNET_OK;
}

// What the matrices of the chain can hold.  They are functions of one variable, the singular value x in [0, 1] that a direction starts with, and the host
// carries intervals of it through the recurrences: the image of an interval under one polynomial is exact (its ends and the polynomial's own extrema), so no
// peak lies between two samples -- with (1.5012, -3.8716, 1.2536) one of 2e8 did between 97 points.  Only the product of the composed factors is bounded as a
// product of intervals, hence the cells; 192 of them, denser towards zero, where singular values grow fastest, overstate it by a few per cent.
constexpr int NS_CELLS = 192;
struct NsSpan { double lo, hi; };
// f over the span: f has no extremum but at the points e
template <typename F> static NsSpan ns_image(const NsSpan& s, const double* e, int n, F f)
{
    const double u = f(s.lo), v = f(s.hi);
    NsSpan r = {u < v ? u : v, u < v ? v : u};
    for (int i = 0; i < n; ++i)
        if (e[i] > s.lo && e[i] < s.hi) { const double w = f(e[i]); r.lo = w < r.lo ? w : r.lo; r.hi = w > r.hi ? w : r.hi; }
    return r;
}
// real roots of p + q s + r s^2
static int ns_roots(double p, double q, double r, double* e)
{
    const double d = q * q - 4.0 * p * r;
    if (!(d >= 0.0)) return 0;
    const double t = -0.5 * (q + (q < 0.0 ? -sqrt(d) : sqrt(d)));
    int n = 0;
    if (r != 0.0) e[n++] = t / r;
    if (t != 0.0) e[n++] = p / t;
    return n;
}
static NsSpan ns_square(const NsSpan& s)
{
    const double u = s.lo * s.lo, v = s.hi * s.hi;
    return NsSpan{s.lo <= 0.0 && s.hi >= 0.0 ? 0.0 : u < v ? u : v, u < v ? v : u};
}
static NsSpan ns_times(const NsSpan& s, const NsSpan& t)
{
    const double v[4] = {s.lo * t.lo, s.lo * t.hi, s.hi * t.lo, s.hi * t.hi};
    return NsSpan{*std::min_element(v, v + 4), *std::max_element(v, v + 4)};
}
// The power-of-two scale of a matrix whose eigenvalues lie in the spans leaves a factor of two below the largest float16.  0: out of range.  (top: of X, which
// a matrix below eps has as X / t, up to 1)
static float ns_scale(const NsSpan* v, double top = 1e-3)
{
    for (int i = 0; i < NS_CELLS; ++i) {
        if (!(v[i].lo >= -4096.0) || !(v[i].hi <= 4096.0)) return 0.f;
        if (-v[i].lo > top) top = -v[i].lo;
        if (v[i].hi > top) top = v[i].hi;
    }
    double s = 1.0;
    while (s * top > 32768.0) s *= 0.5;
    while (s * top * 2.0 <= 32768.0) s *= 2.0;
    return (float)s;
}

// The launches behind the pack pass
struct NsOp { int apply, ny; NsProds pr; int q, xt; float alpha, beta; bool gram, last; float grown, grown_to; };      // grown: NsView::t
struct NsSchedule { int count; float sx; NsOp op[32 * 4]; };

// first, later: steps composed at once in the first block and in the others (see the head of this file).  False: the coefficients drive singular values
// out of range
static bool ns_build_schedule(const saunet_ns_desc* d, int first, int later, NsSchedule& w)
{
    NsSpan X[NS_CELLS], S[NS_CELLS], P[NS_CELLS], T[NS_CELLS], V[NS_CELLS];
    const double a0 = d->a, b = d->b, c = d->c;
    for (int i = 0; i < NS_CELLS; ++i) {
        const double u = (double)i / NS_CELLS, v = (double)(i + 1) / NS_CELLS;
        X[i] = NsSpan{u * u * u * u, v * v * v * v * (1.0 + 1e-6)};
    }
    // extrema of b s + c s^2, of s (a + b s + c s^2) and, in x, of x (a + b x^2 + c x^4)
    double ep[1], er[2], ex[4];
    const int np = c != 0.0 ? (ep[0] = -b / (2.0 * c), 1) : 0, nr = ns_roots(a0, 2.0 * b, 3.0 * c, er);
    int nx = ns_roots(a0, 3.0 * b, 5.0 * c, ex);
    for (int i = 0, n = nx; i < n; ++i) { ex[i] = sqrt(ex[i]); ex[nx++] = -ex[i]; }           // (a NaN lies in no span)
    float sx = w.sx = ns_scale(X);
    w.count = 0;
    int xt = 0;
    float grown = 1.f;
    auto push = [&](int ny, const NsProds& pr, bool gram) { w.op[w.count++] = NsOp{0, ny, pr, 0, 0, 0.f, 0.f, gram, false, grown, 1.f}; };
    for (int done = 0; done < d->steps;) {
        const int left = d->steps - done, most = done ? later : first, nb = left < most ? left : most;
        // P is kept as b S + c S^2 in the first block, where most s are small, and as that + (a - 1) I, near zero where s is near 1, later: its rounding
        // counts in units of what is kept (300 x 500, five steps: 3.1e-6 of |X| without the shift, 1.6e-6 with it)
        const double a = done ? 1.0 : a0, shift = a0 - a;
        for (int i = 0; i < NS_CELLS; ++i) S[i] = ns_square(X[i]);
        float sa = ns_scale(S), sp, sq = 0;
        if (sa == 0.f) return false;
        push(1, NsProds{{{NS_X, NS_X, -1, -1, NS_A, sa / (sx * sx), 0.f, 0.f}, {}}}, true);
        double q = 0;
        int Qb = NS_Q0;
        for (int j = 0; j < nb; ++j) {
            for (int i = 0; i < NS_CELLS; ++i) P[i] = ns_image(S[i], ep, np, [&](double s) { return (c * s + b) * s + shift; });
            sp = ns_scale(P);
            if (sp == 0.f) return false;
            const int Pb = j ? NS_P : NS_Q0;
            push(1, NsProds{{{NS_A, NS_A, NS_A, -1, Pb, (float)(c * sp / ((double)sa * sa)), (float)(b * sp / sa), 0.f, (float)(shift * sp)}, {}}}, false);
            NsProds pr = {};
            int ny = 0;
            // T: the product of the factors a + P so far; what is kept of it is T - q I
            if (j == 0) { for (int i = 0; i < NS_CELLS; ++i) T[i] = NsSpan{P[i].lo + a, P[i].hi + a}; sq = sp; q = a; }
            else {
                for (int i = 0; i < NS_CELLS; ++i) {
                    T[i] = ns_times(T[i], NsSpan{P[i].lo + a, P[i].hi + a});
                    V[i] = NsSpan{T[i].lo - q * a, T[i].hi - q * a};
                }
                const float s2 = ns_scale(V);
                if (s2 == 0.f) return false;
                const int to = Qb == NS_Q0 ? NS_Q1 : NS_Q0;
                pr.p[ny++] = {NS_P, Qb, Qb, NS_P, to, (float)(s2 / ((double)sp * sq)), (float)(a * s2 / sq), (float)(q * s2 / sp)};
                Qb = to; sq = s2; q *= a;
            }
            float sr = 0;
            if (j < nb - 1) {
                for (int i = 0; i < NS_CELLS; ++i) V[i] = ns_image(S[i], er, nr, [&](double s) { return ((c * s + b) * s + a0) * s; });
                sr = ns_scale(V);
                if (sr == 0.f) return false;
                pr.p[ny++] = {Pb, NS_A, NS_A, -1, NS_R, (float)(sr / ((double)sp * sa)), (float)(a * sr / sa), 0.f};
            }
            if (ny) push(ny, pr, false);
            for (int i = 0; i < NS_CELLS; ++i) X[i] = ns_image(X[i], ex, nx, [&](double x) { return ((c * x * x + b) * x * x + a0) * x; });
            if (j < nb - 1) {
                for (int i = 0; i < NS_CELLS; ++i) S[i] = ns_square(X[i]);
                const float s2 = ns_scale(S);
                if (s2 == 0.f) return false;
                push(1, NsProds{{{NS_R, Pb, NS_R, -1, NS_A, (float)(s2 / ((double)sr * sp)), (float)(a * s2 / sr), 0.f}, {}}}, false);
                sa = s2;
            }
        }
        done += nb;
        const bool last = done >= d->steps;
        const float s2 = last ? 1.f : ns_scale(X, 1.0);
        if (s2 == 0.f) return false;
        double growth = 1.0;
        for (int i = 0; i < NS_CELLS; ++i) while (T[i].hi > growth || -T[i].lo > growth) growth *= 2.0;
        const float to = grown * growth < 0x1p126 ? (float)(grown * growth) : 0x1p126f;
        w.op[w.count++] = NsOp{1, 0, {}, Qb, xt, (float)(s2 / ((double)sq * sx)), (float)(q * s2 / sx), false, last, grown, to};
        xt ^= 1; sx = s2; grown = to;
    }
    return true;
}
// The schedule is a function of the numbers below alone and costs some 50 us of host time, so a thread keeps the last few: an optimiser asks for the same
// one or two in every step
static const NsSchedule* ns_schedule(const saunet_ns_desc* d, int first, int later)
{
    struct Key { float a, b, c; int steps, first, later; };
    struct Entry { Key key; bool ok; NsSchedule w; };
    static thread_local Entry kept[4];
    static thread_local int next = 0;
    const Key k = {d->a, d->b, d->c, d->steps, first, later};
    for (Entry& e : kept) if (e.key.steps && !memcmp(&e.key, &k, sizeof k)) return e.ok ? &e.w : nullptr;
    Entry& e = kept[next];
    next = (next + 1) & 3;
    e.key = k;
    e.ok = ns_build_schedule(d, first, later, e.w);
    return e.ok ? &e.w : nullptr;
}

template <class Core, typename T, int MODE> static void ns_launch_apply(const saunet_ns_desc* d, const NsPlan& p, const NsTable& tab, const NsOp& o, const float* hyper, hipStream_t st)
{
    static DeviceOnce once;
    once.lds((const void*)ns_apply_kernel<Core, T, MODE>, Core::LDS);
    hipLaunchKernelGGL((ns_apply_kernel<Core, T, MODE>), dim3(ns_deal_grid(p.deal[NS_KINDS])), dim3(Core::NT), Core::LDS, st, tab, o.q, o.xt, o.alpha, o.beta, o.grown, o.grown_to, hyper, d->adjust, p.deal[NS_KINDS]);
}
template <class Core> static void ns_launch_prod(const NsPlan& p, const NsTable& tab, const NsOp& o, hipStream_t st)
{
    const int kind = o.gram ? NS_GRAM : o.ny == 2 ? NS_TWO : NS_ONE;
    static DeviceOnce once;
    once.lds((const void*)ns_prod_kernel<Core>, Core::LDS);
    const unsigned dealt = ns_deal_grid(p.deal[kind]);
    hipLaunchKernelGGL((ns_prod_kernel<Core>), dim3(dealt + (unsigned)(p.grid[kind] - p.deal[kind].b[8]), o.ny), dim3(Core::NT), Core::LDS, st, tab, kind, o.pr, o.grown, p.deal[kind], (int)dealt);
    if constexpr (Core::KW == 1) if (p.cut[kind]) hipLaunchKernelGGL((ns_finish_kernel<Core>), dim3((unsigned)(p.cut[kind] * NsQuads<Core>::N), o.ny), dim3(Core::NT), 0, st, tab, kind, o.pr, o.grown);
}

// The matrices with up to NS_MID rows and the others are two chains of launches: the short ones go step by step and keep the digits that composing would cost
// them.  A Muon step does not need those -- its result is multiplied by the learning rate and added to a rounded parameter -- so there a list with both
// goes through one chain (SAUNet's matrices 936 us, in two chains 1090).  k: 0 the short ones, 1 the others
constexpr int NS_MID = 128;
static saunet_ns_desc ns_part(const saunet_ns_desc* d, bool muon, int k, saunet_ns_item* item)
{
    saunet_ns_desc r = *d;
    r.item = item; r.count = 0;
    if (muon)
        for (int i = 0; i < d->count; ++i)
            if ((d->item[i].rows < d->item[i].cols ? d->item[i].rows : d->item[i].cols) > NS_MID) { r.item = d->item; r.count = k == 1 ? d->count : 0; return r; }
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        if (((t.rows < t.cols ? t.rows : t.cols) > NS_MID) == (k == 1)) item[r.count++] = t;
    }
    return r;
}

// A list goes through the chain in parts of so many bytes of workspace, one behind the other in the same memory (a part holds one matrix at least): X, two
// of X^T and five m x m matrices for each would come to eight times the parameters of a square one.  ms a call with parts of 1, 2, 4, 16 GiB: forty 2048 x 2048
// 24.0, 23.7, 23.6, 23.4; sixty 512 x 13824 8.8, 8.0, 7.8, 7.8; 1500 of 256 x 1024 11.7, 11.2, 11.2, 10.9; nine 4096 x 11008 56.9, 59.7, 59.0, 59.3.
constexpr long NS_PART = 4L << 30;
// how many of the matrices from `from` on make the next part
static int ns_next(const saunet_ns_desc* d, int from)
{
    long sum = 0;
    for (int i = from; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        const long elements = (long)t.rows * t.cols, cols = ((t.rows < t.cols ? t.cols : t.rows) + NSS_COLS - 1) / NSS_COLS;
        sum += ns_is_small(d, t) ? (1 + (cols < 64 ? cols : 64)) * 8192 : NsView::bytes(t.rows, t.cols) + elements / (NS_NORM / 8);
        if (sum > NS_PART && i > from) return i - from;
    }
    return d->count - from;
}
// fn(part) for every part of either chain until one returns an error
template <typename F> static int ns_parts(const saunet_ns_desc* d, bool muon, saunet_ns_item* item, F fn)
{
    for (int k = 0; k < 2; ++k) {
        const saunet_ns_desc chain = ns_part(d, muon, k, item);
        for (int at = 0, n; at < chain.count; at += n) {
            saunet_ns_desc part = chain;
            part.item += at;
            part.count = n = ns_next(&chain, at);
            const int rc = fn(part);
            if (rc) return rc;
        }
    }
    return SAUNET_OK;
}

// Steps composed at once: see the head of this file.  The longest matrix is the first.  (Short ones in twos would gain little, measured with 64 x 64
// tiles: one of 128 x 256 183 us, step by step 171; sixty of 128 x 64 .. 992 299 us against 324.)
static const NsSchedule* ns_plan_schedule(const saunet_ns_desc* d, bool muon, const NsPlan& p, const NsItem* large)
{
    const bool compose = p.large && (large[0].rows < large[0].cols ? large[0].rows : large[0].cols) > NS_MID && p.shortest > 32 && (double)d->a * d->a <= 16.0;
    return ns_schedule(d, !compose ? 1 : !muon && p.shortest < 256 ? 2 : 3, compose ? 2 : 1);
}

// go: false looks only whether the call can be made
template <typename T, bool MUON> static int ns_run(const saunet_ns_desc* d, bool go, const float* hyper, void* workspace, int64_t workspace_bytes, hipStream_t st, const char* who)
{
    static thread_local NsItem large[4096];
    static thread_local NssItem small[4096];
    NsPlan p;
    char* ws = (char*)workspace;
    int rc = ns_plan(d, p, large, small, ws);
    if (rc) return rc;
    if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255)) return set_error(SAUNET_BAD_SHAPE, "%s: the workspace has to hold %ld bytes on a 256-byte border", who, p.bytes);
    const NsSchedule* w = ns_plan_schedule(d, MUON, p, large);
    if (!w) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
    if (!go) return SAUNET_OK;
    for (long i = 0; i < p.small; i += NSS_CHUNK) {
        NssItems ch;
        const int k = (int)(p.small - i < NSS_CHUNK ? p.small - i : NSS_CHUNK);
        int grid = 0;
        ch.ws = (double*)(ws + p.small_at);
        for (int j = 0; j < k; ++j) { ch.it[j] = small[i + j]; ch.it[j].p = grid; grid += small[i + j].p; }
        p.small_at += (long)(grid + k) * 1024 * 8;
        hipLaunchKernelGGL((nss_gram_kernel<T, MUON>), dim3(grid), dim3(256), 0, st, ch, k, hyper);
        hipLaunchKernelGGL(nss_poly_kernel, dim3(k), dim3(512), 0, st, ch, d->steps, (double)d->a, (double)d->b, (double)d->c, d->eps);
        hipLaunchKernelGGL((nss_apply_kernel<T, MUON>), dim3(grid), dim3(256), 0, st, ch, k, hyper, d->adjust);
        SAUNET_CHECK_LAUNCH("nss_apply");
    }
    if (!p.large) return SAUNET_OK;
    const NsTable tab = {(const NsItem*)(ws + p.tab_at), (int)p.large, large[0]};
    double* part = (double*)(ws + p.part_at);
    const int n = (int)p.large;
    for (int i = 0; n > 1 && i < n; i += NS_CHUNK) {
        NsItems ch;
        const int k = n - i < NS_CHUNK ? n - i : NS_CHUNK;
        memcpy(ch.it, large + i, sizeof(NsItem) * k);
        hipLaunchKernelGGL(ns_setup_kernel, dim3(1), dim3(64), 0, st, ch, k, (NsItem*)tab.all + i);
    }
    hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)p.norm), dim3(256), 0, st, tab, hyper, part);
    hipLaunchKernelGGL((ns_pack_kernel<T, MUON>), dim3((unsigned)p.pack), dim3(256), 0, st, tab, hyper, part, d->eps, w->sx);
    SAUNET_CHECK_LAUNCH("ns_pack");
    for (int i = 0; i < w->count; ++i) {
        const NsOp& o = w->op[i];
        if (o.apply) {
            constexpr int LAST = MUON ? 2 : 1;
            if (p.tile_n == 32) o.last ? ns_launch_apply<NsCore32, T, LAST>(d, p, tab, o, hyper, st) : ns_launch_apply<NsCore32, T, 0>(d, p, tab, o, hyper, st);
            else if (p.tile_n == 64) o.last ? ns_launch_apply<NsCore64, T, LAST>(d, p, tab, o, hyper, st) : ns_launch_apply<NsCore64, T, 0>(d, p, tab, o, hyper, st);
            else o.last ? ns_launch_apply<NsCore128, T, LAST>(d, p, tab, o, hyper, st) : ns_launch_apply<NsCore128, T, 0>(d, p, tab, o, hyper, st);
            SAUNET_CHECK_LAUNCH("ns_apply");
        } else {
            const int kind = o.gram ? NS_GRAM : o.ny == 2 ? NS_TWO : NS_ONE;
            if ((o.gram ? p.tile_g : p.tile_m) == 32) ns_launch_prod<NsCore32>(p, tab, o, st);
            else if ((o.gram ? p.tile_g : p.tile_m) == 64) ns_launch_prod<NsCore64>(p, tab, o, st);
            else if (p.grid[kind] * o.ny <= NS_SLOTS / 2) ns_launch_prod<NsCore128W>(p, tab, o, st);
            else ns_launch_prod<NsCore128>(p, tab, o, st);
            SAUNET_CHECK_LAUNCH("ns_prod");
        }
    }
    return SAUNET_OK;
}

template <typename T, bool MUON> static int ns_run_all(const saunet_ns_desc* d, const float* hyper, void* workspace, int64_t workspace_bytes, hipStream_t st, const char* who)
{
    static thread_local saunet_ns_item item[4096];
    for (int pass = 0; pass < 2; ++pass) {
        const int rc = ns_parts(d, MUON, item, [&](const saunet_ns_desc& part) { return ns_run<T, MUON>(&part, pass == 1, hyper, workspace, workspace_bytes, st, who); });
        if (rc) return rc;
    }
    return SAUNET_OK;
}

}  // namespace saunet

using namespace saunet;

extern "C" {

int64_t saunet_newton_schulz_workspace(const saunet_ns_desc* d)
{
    static thread_local NsItem large[4096];
    static thread_local NssItem small[4096];
    static thread_local saunet_ns_item item[4096];
    NsPlan p;
    int rc = ns_check(d, "newton_schulz");
    int64_t most = 0;
    bool bad[2] = {false, false};                 // a use whose schedules leave the range: the step composes otherwise than the plain call
    for (int use = 0; use < 2 && !rc; ++use)
        rc = ns_parts(d, use == 1, item, [&](const saunet_ns_desc& part) {
            const int status = ns_plan(&part, p, large, small, nullptr);
            if (status) return status;
            if (p.bytes > most) most = p.bytes;
            if (!ns_plan_schedule(&part, use == 1, p, large)) bad[use] = true;
            return (int)SAUNET_OK;
        });
    if (!rc && bad[0] && bad[1]) return set_error(SAUNET_UNSUPPORTED, "newton_schulz: the coefficients drive singular values out of range");
    return rc ? rc : most;
}

int saunet_newton_schulz(const saunet_ns_desc* d, void* workspace, int64_t workspace_bytes, void* stream)
{
    int rc = ns_check(d, "newton_schulz");
    if (rc) return rc;
    for (int i = 0; i < d->count; ++i) if (!d->item[i].src || !d->item[i].dst) return set_error(SAUNET_BAD_SHAPE, "newton_schulz: matrix %d has no memory", i);
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == SAUNET_F32) return ns_run_all<float, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
    if (d->dtype == SAUNET_BF16) return ns_run_all<u16, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
    return ns_run_all<_Float16, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
}

int saunet_muon_step(const saunet_ns_desc* d, const float* hyper, void* workspace, int64_t workspace_bytes, void* stream)
{
    int rc = ns_check(d, "muon");
    if (rc) return rc;
    if (d->dtype != SAUNET_F32) return set_error(SAUNET_BAD_DTYPE, "muon: parameters, gradients and momentum are float32");
    if (!hyper) return set_error(SAUNET_BAD_SHAPE, "muon: no hyper-parameters");
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        if (!t.src || !t.dst || !t.buf) return set_error(SAUNET_BAD_SHAPE, "muon: matrix %d has no memory", i);
        if (t.ld_src != t.cols || t.ld_dst != t.cols) return set_error(SAUNET_BAD_SHAPE, "muon: matrix %d is not contiguous", i);
    }
    return ns_run_all<float, true>(d, hyper, workspace, workspace_bytes, (hipStream_t)stream, "muon");
}

}  // extern "C"
