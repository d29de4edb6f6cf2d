// Matrix products of int8 rows: y[m][n] = (sum_k a[m][k] b[n][k]) sa[m] sb[n] + bias[n], optionally clamped at zero, and the quantisation of
// floating-point rows that feeds them.
//
//   quantise   s = fl32(max |x| / 127),  q = round-half-even(x / s)  with the EXACT quotient, so q is a function of the row alone
//
// The integer sums are exact (K <= 131071 keeps them inside 32 bits); float32 enters with the two scales and the bias, one rounding to the output type at
// the end.  Rows are padded with zeros to a multiple of 64 bytes, so the reduction has no tail.
#include "nt_tiles.h"

namespace saunet {

typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

template <typename T> struct QElem;
template <> struct QElem<float> {
    static constexpr int V = 4;          // elements of a 16-byte vector
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { Vec16<float>::unpack(v, f); }
};
template <> struct QElem<u16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ float load(const u16* p) { return Elem<u16>::load(p); }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { Vec16<u16>::unpack(v, f); }
};
template <> struct QElem<_Float16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f)
    {
        const f16x8_t h = __builtin_bit_cast(f16x8_t, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
    }
};

struct QScale { float s, inv; };
// from the bits of the largest magnitude: a row with an Inf or NaN gets scale NaN and zeros (its products are NaN); a row whose scale would be
// subnormal counts as zero
__device__ __forceinline__ QScale q_scale(unsigned top)
{
    QScale r;
    r.s = __uint_as_float(top) / 127.f;
    if (top >= 0x7f800000u) { r.s = __uint_as_float(0x7fc00000u); r.inv = 0.f; }
    else if (r.s < 1.17549435e-38f) { r.s = 0.f; r.inv = 0.f; }
    else r.inv = 1.f / r.s;
    return r;
}
// round-half-even of the exact x / s.  x * inv is within 2^-16 of it, so its rounding is off by one at most and only beside a half; x - q s is exact
// in float32 (a multiple of the finer of two neighbouring units, no larger than s), so the comparison with s / 2 settles it.
__device__ __forceinline__ int q_round(float x, const QScale& s)
{
    if (!(s.inv > 0.f)) return 0;
    float q = rintf(x * s.inv);
    const float e = fmaf(-q, s.s, x), t = 2.f * fabsf(e);
    if (t > s.s || (t == s.s && ((int)q & 1))) q += e > 0.f ? 1.f : -1.f;
    return (int)q;
}

// four of them as bytes.  x * inv + 1.5 * 2^23 rounds half to even in its last place and holds q in its low byte; only a quotient within rounding of a
// half takes the exact path.
__device__ __forceinline__ unsigned q_round4(const float* x, const QScale& s)
{
    unsigned w[4];
    bool close = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float t = fmaf(x[j], s.inv, 12582912.f);
        close |= fabsf(fmaf(-(t - 12582912.f), s.s, x[j])) >= 0.49999f * s.s;
        w[j] = __float_as_uint(t);
    }
    if (close || !(s.inv > 0.f)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (unsigned)q_round(x[j], s);
    }
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x00000400u), __builtin_amdgcn_perm(w[1], w[0], 0x00000400u), 0x05040100u);
}

struct QArgs { const void* x; long ldx; long rows; int k; const float* scale; const float* shift; int relu; signed char* q; long ldq; float* s; int vec; };

// the largest of `top` over the G lanes of a row (256: the workgroup)
template <int G> __device__ __forceinline__ unsigned q_top(unsigned top)
{
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) { const unsigned b = __shfl_xor(top, o, 64); top = b > top ? b : top; }
    if (G == 256) {
        __shared__ unsigned s_top[4];
        if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) top = s_top[w] > top ? s_top[w] : top;
    }
    return top;
}

// G lanes a row, NV vectors a lane kept in registers (k <= G * NV * V, 16-byte aligned rows); NV == 0: any k and alignment, the row is read twice
// PRO: scale / shift / relu in front (16-byte aligned vectors where NV > 0)
template <typename T, int G, int NV, bool PRO> __global__ __launch_bounds__(256) void quantize_rows_kernel(QArgs a)
{
    constexpr int V = QElem<T>::V;
    const int lane = threadIdx.x % G;
    const long row = (long)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= a.rows) return;                                       // whole groups leave together
    const T* x = (const T*)a.x + row * a.ldx;
    signed char* q = a.q + row * a.ldq;
    auto pro = [&](float v, int c) { if (a.scale) { v = fmaf(v, a.scale[c], a.shift[c]); } return a.relu && v < 0.f ? 0.f : v; };
    unsigned top = 0;
    if (NV > 0) {
        float f[NV ? NV : 1][V];
        u32x4 v[NV ? NV : 1];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            v[i] = u32x4{0u, 0u, 0u, 0u};
            if (c + V <= a.k) v[i] = *(const u32x4*)(x + c);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            QElem<T>::unpack(v[i], f[i]);
            if (c < a.k && c + V > a.k) for (int j = 0; j < V; ++j) f[i][j] = c + j < a.k ? QElem<T>::load(x + c + j) : 0.f;
            if (PRO && c + V <= a.k) {
                if (a.scale)
#pragma unroll
                    for (int h = 0; h < V; h += 4) {
                        const f32x4 sc = *(const f32x4*)(a.scale + c + h), sh = *(const f32x4*)(a.shift + c + h);
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[i][h + j] = fmaf(f[i][h + j], sc[j], sh[j]);
                    }
                if (a.relu)
#pragma unroll
                    for (int j = 0; j < V; ++j) f[i][j] = f[i][j] < 0.f ? 0.f : f[i][j];
            } else if (PRO) {
                for (int j = 0; j < V; ++j) if (c + j < a.k) f[i][j] = pro(f[i][j], c + j);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) { const unsigned b = __float_as_uint(f[i][j]) & 0x7fffffffu; top = b > top ? b : top; }
        }
        const QScale s = q_scale(q_top<G>(top));
        if (lane == 0) a.s[row] = s.s;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            if (c >= a.ldq) continue;
            if (V == 8) *(u32x2*)(q + c) = u32x2{q_round4(f[i], s), q_round4(f[i] + (V == 8 ? 4 : 0), s)};
            else *(unsigned*)(q + c) = q_round4(f[i], s);
        }
        for (int c = (NV * G + lane) * V; c < a.ldq; c += G * V) {       // padding beyond the registers' reach
            if (V == 8) *(u32x2*)(q + c) = u32x2{0u, 0u};
            else *(unsigned*)(q + c) = 0u;
        }
    } else {
        for (int c = lane; c < a.k; c += G) { const unsigned b = __float_as_uint(pro(QElem<T>::load(x + c), c)) & 0x7fffffffu; top = b > top ? b : top; }
        const QScale s = q_scale(q_top<G>(top));
        if (lane == 0) a.s[row] = s.s;
        for (int c = lane * 4; c < a.ldq; c += G * 4) {
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = c + j < a.k ? pro(QElem<T>::load(x + c + j), c + j) : 0.f;
            *(unsigned*)(q + c) = q_round4(f, s);
        }
    }
}

// Lanes a row: as few as hold it in one or two vectors each, so that a wave keeps several short rows in flight; a workgroup to a row where there are
// fewer rows than would fill the card with a wave each
template <typename T, bool PRO> static void q_launch(const QArgs& a, hipStream_t st)
{
    constexpr int V = QElem<T>::V;
#define Q_GO(G, NV) hipLaunchKernelGGL((quantize_rows_kernel<T, G, NV, PRO>), dim3((unsigned)((a.rows + 256 / G - 1) / (256 / G))), dim3(256), 0, st, a)
    const bool few = a.rows <= 1024 && a.k > 128 * V;
    if (!a.vec || a.k > 2048 * V) { if (a.rows <= 4096 && a.k > 256) Q_GO(256, 0); else Q_GO(64, 0); }
    else if (a.k <= 16 * V) Q_GO(16, 1);
    else if (a.k <= 32 * V) Q_GO(16, 2);
    else if (a.k <= 64 * V) Q_GO(64, 1);
    else if (a.k <= 128 * V) Q_GO(64, 2);
    else if (a.k <= 256 * V) { if (few) Q_GO(256, 1); else Q_GO(64, 4); }
    else if (a.k <= 512 * V) { if (few) Q_GO(256, 2); else Q_GO(64, 8); }
    else if (a.k <= 1024 * V) Q_GO(256, 4);
    else Q_GO(256, 8);
#undef Q_GO
}

// ---- the product ------------------------------------------------------------------------------------------------------------------
struct I8Args { const char* a; const float* sa; long lda; long m; const char* b; const float* sb; long ldb; int n; int ksteps; const float* bias; int relu; void* y; long ldy; int vec; int tn; };

template <typename T> struct YElem;
template <> struct YElem<float> { typedef f32x4 V4; static __device__ __forceinline__ float cvt(float v) { return v; } };
template <> struct YElem<u16> { typedef __attribute__((ext_vector_type(4))) u16 V4; static __device__ __forceinline__ u16 cvt(float v) { return __builtin_bit_cast(u16, (__bf16)v); } };
template <> struct YElem<_Float16> { typedef __attribute__((ext_vector_type(4))) _Float16 V4; static __device__ __forceinline__ _Float16 cvt(float v) { return (_Float16)v; } };

// Operand A of the MFMA is the WEIGHT tile (BM channels), operand B the token tile (BN tokens): a lane then holds four consecutive channels of one token.
// The wave's 32 tokens x (BM / WGM) channels go through LDS so that the stores are whole rows of the tile.
template <typename T, class Core> __global__ __launch_bounds__(Core::NT) void matmul_int8_kernel(I8Args g)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    int tt, tc;
    nt_band(nt_xcd(blockIdx.x, gridDim.x), (int)((g.m + Core::BN - 1) / Core::BN), g.tn, tt, tc);
    const long m0 = (long)tt * Core::BN;
    const int n0 = tc * Core::BM;
    typename Core::Acc acc[Core::TM][Core::TN] = {};
    const long ml = g.m - m0;
    Core::run(g.b + (long)n0 * g.ldb, (unsigned)g.ldb, g.n - n0, g.a + m0 * g.lda, (unsigned)g.lda, ml < Core::BN ? (int)ml : Core::BN, g.ksteps, smem, acc);
    __syncthreads();
    constexpr int CH = Core::BM / Core::WGM, PITCH = CH * (int)sizeof(T) + 16;          // one wave: 32 tokens of CH channels
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / Core::WGN, wn = wave % Core::WGN, half = lane >> 5, tok = lane & 31;
    float* s_sb = (float*)smem;
    float* s_bias = s_sb + Core::BM;
    for (int c = threadIdx.x; c < Core::BM; c += Core::NT) {
        const int n = n0 + c < g.n ? n0 + c : g.n - 1;
        s_sb[c] = g.sb[n];
        s_bias[c] = g.bias ? g.bias[n] : 0.f;
    }
    __syncthreads();
    unsigned char* buf = smem + Core::BM * 8 + wave * 32 * PITCH;
    const int nw = n0 + wm * CH;
#pragma unroll
    for (int tj = 0; tj < Core::TN; ++tj) {
        const long mt = m0 + wn * (Core::BN / Core::WGN) + tj * 32;
        const float sa = mt + tok < g.m ? g.sa[mt + tok] : 0.f;
#pragma unroll
        for (int ti = 0; ti < Core::TM; ++ti)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = ti * 32 + q * 8 + half * 4;
                const f32x4 sb = *(const f32x4*)(s_sb + wm * CH + c), bias = *(const f32x4*)(s_bias + wm * CH + c);
                typename YElem<T>::V4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = fmaf((float)acc[ti][tj][q * 4 + r] * sa, sb[r], bias[r]);
                    if (g.relu && v < 0.f) v = 0.f;
                    o[r] = YElem<T>::cvt(v);
                }
                *(typename YElem<T>::V4*)(buf + tok * PITCH + c * sizeof(T)) = o;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own rows: no other wave reads them
        constexpr int VPR = CH * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T);
        for (int k = lane; k < 32 * VPR; k += 64) {
            const int t = k / VPR, c = (k % VPR) * E;
            if (mt + t >= g.m || nw + c >= g.n) continue;
            const u32x4 v = *(const u32x4*)(buf + t * PITCH + c * sizeof(T));
            T* y = (T*)g.y + (mt + t) * g.ldy + nw + c;
            if (g.vec && nw + c + E <= g.n) *(u32x4*)y = v;
            else {
                const T* o = (const T*)(buf + t * PITCH + c * sizeof(T));
                for (int j = 0; j < E && nw + c + j < g.n; ++j) y[j] = o[j];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Tile by the amount of work, counted in 64 x 64 tiles (bf16 out; us for channels x tokens of a tile, K the reduction; L: four stages instead of two):
//                                    64x64  128x64  128x128  128x128L  256x256
//   8192 x 4096, K 4096  (8192 tiles)   276     234      178       179      142      a long reduction and work for every CU: operand traffic is the bound
//   131072 x 128, K 256  (4096 tiles)  21.1    18.2     16.3      18.9     27.9      a short one: memory is, several workgroups a CU overlap loads and stores
//   4096 x 1024, K 8192  (1024 tiles)    80      65       55        50      101
//   2048 x 2048, K 2048  (1024 tiles)  22.4    19.7     15.5      15.8     33.5
//   8192 x 256, K 8192    (512 tiles)  42.6    33.2     49.8      40.8      101      too few large tiles to fill the card: the smallest that do
//   512 x 512, K 512       (64 tiles)   4.4     5.4      5.7       6.2     14.1
// Where one side is short a wide tile multiplies rows that do not exist.  Up to 64 the smallest tile wins whatever the work, the largest one from some 192 on:
//   200000 x 8, K 1024                 34.1    49.6      42.6      45.4     88.5
//   60000 x 40, K 2048                 22.3    28.7      23.1      24.3     38.2
//   64 x 200000, K 1024                37.0    37.1      45.0      46.0     86.7
//   200000 x 65, K 1024                75.5    59.5      59.6      65.2      104
//   200000 x 160, K 1024               86.9    96.4      81.9      84.2     93.6
//   200000 x 200, K 1024                124     107      95.5      95.5      100
typedef NtCore<NtI8, 64, 64, 2, 2, 4> I8Core64;
typedef NtCore<NtI8, 128, 64, 2, 2, 4> I8CoreTall;
typedef NtCore<NtI8, 128, 128, 2, 4, 2> I8Core128;
typedef NtCore<NtI8, 128, 128, 4, 2, 4> I8Core128L;
typedef NtCore<NtI8, 256, 256, 2, 4, 4> I8Core256;

template <typename T, class Core> static int mm8_tiles(I8Args g, hipStream_t st)
{
    constexpr int EPI = Core::BM * 8 + Core::NW * 32 * (Core::BM / Core::WGM * (int)sizeof(T) + 16), LDS = Core::LDS > EPI ? Core::LDS : EPI;
    static_assert(LDS <= 160 * 1024, "the wave's rows fit");
    static DeviceOnce once;
    once.lds((const void*)matmul_int8_kernel<T, Core>, LDS);
    g.tn = cdiv(g.n, Core::BM);
    const long tiles = (g.m + Core::BN - 1) / Core::BN * g.tn;
    if (tiles > 0xffffffffL / Core::NT) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: %ld rows of %d channels are too much for one launch", g.m, g.n);
    hipLaunchKernelGGL((matmul_int8_kernel<T, Core>), dim3((unsigned)tiles), dim3(Core::NT), LDS, st, g);
    SAUNET_CHECK_LAUNCH("matmul_int8");
    return SAUNET_OK;
}

// ---- few tokens or channels: the operands go straight into registers -------------------------------------------------------------------------
// A workgroup owns 16 channels and MT x 16 tokens; its 8 waves take the 64-byte steps of the reduction in turn, mfma_i32_16x16x64_i8 with 16 weight rows
// against the tokens, and add their sums through LDS. 
constexpr int FEW_WAVES = 8, FEW_UNROLL = 8;

template <typename T, int MT> __global__ __launch_bounds__(FEW_WAVES * 64) void matmul_int8_few_kernel(I8Args g)
{
    __shared__ int s_red[FEW_WAVES][MT][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kq = (lane >> 4) * 16;
    const int n0 = blockIdx.x * 16;
    const long m0 = (long)blockIdx.y * MT * 16;
    const char* b = g.b + (long)(n0 + r < g.n ? n0 + r : g.n - 1) * g.ldb + kq;
    const char* a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) { const long m = m0 + t * 16 + r; a[t] = g.a + (m < g.m ? m : g.m - 1) * g.lda + kq; }
    i32x4 acc[MT] = {};
    for (int s0 = wave; s0 < g.ksteps; s0 += FEW_WAVES * FEW_UNROLL) {
        i32x4 fb[FEW_UNROLL];
#pragma unroll
        for (int u = 0; u < FEW_UNROLL; ++u) { const int s = s0 + u * FEW_WAVES; fb[u] = s < g.ksteps ? __builtin_nontemporal_load((const i32x4*)(b + (long)s * 64)) : i32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int u = 0; u < FEW_UNROLL; ++u) {
            const int s = s0 + u * FEW_WAVES;
            if (s >= g.ksteps) break;
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u], *(const i32x4*)(a[t] + (long)s * 64), acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_red[wave][t][r][(lane >> 4) * 4 + i] = acc[t][i];
    __syncthreads();
    for (int k = threadIdx.x; k < MT * 256; k += FEW_WAVES * 64) {
        const int c = k & 15, t = k >> 4, n = n0 + c;
        const long m = m0 + t;
        if (m >= g.m || n >= g.n) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) sum += s_red[w][t >> 4][t & 15][c];
        float v = fmaf((float)sum * g.sa[m], g.sb[n], g.bias ? g.bias[n] : 0.f);
        if (g.relu && v < 0.f) v = 0.f;
        ((T*)g.y)[m * g.ldy + n] = YElem<T>::cvt(v);
    }
}

// The same for up to 8 floating-point rows: every workgroup quantises all of them into LDS, 512 / (rows rounded up to a power of two) threads a row,
// while its first weight loads are in flight.  One launch instead of two, us: one row of 4096 through 4096 channels 7.7 against 9.1, of 1024 through 512
// 4.1 against 5.4; two rows of 2048 5.9 against 6.2.  Re-quantising in every workgroup costs more than the second launch beyond some 4096 values in
// several rows: two of 4096 9.6 against 9.0, eight of 2048 13.2 against 6.7.
constexpr int FEW_LDS = 16384;

template <typename X, typename T> __global__ __launch_bounds__(FEW_WAVES * 64) void linear_int8_few_kernel(I8Args g, QArgs q, int group)
{
    __shared__ __attribute__((aligned(16))) signed char s_q[FEW_LDS];
    __shared__ int s_red[FEW_WAVES][16][17];
    __shared__ unsigned s_top[FEW_WAVES];
    __shared__ float s_sa[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, kq = (lane >> 4) * 16, n0 = blockIdx.x * 16;
    const char* b = g.b + (long)(n0 + r < g.n ? n0 + r : g.n - 1) * g.ldb + kq;
    i32x4 fb[FEW_UNROLL];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int u = 0; u < FEW_UNROLL; ++u) { const int s = s0 + u * FEW_WAVES; fb[u] = s < g.ksteps ? __builtin_nontemporal_load((const i32x4*)(b + (long)s * 64)) : i32x4{0, 0, 0, 0}; }
    };
    fetch(wave);
    {
        const int row = tid / group, at = tid % group;
        const bool mine = row < q.rows;
        const X* x = (const X*)q.x + (mine ? row : 0) * q.ldx;
        unsigned top = 0;
        if (mine)
            for (int c = at; c < q.k; c += group) { const unsigned t = __float_as_uint(QElem<X>::load(x + c)) & 0x7fffffffu; top = t > top ? t : top; }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { const unsigned t = __shfl_xor(top, o, 64); top = t > top ? t : top; }
        if (lane == 0) s_top[wave] = top;
        __syncthreads();
        const int w0 = wave / (group / 64) * (group / 64);
        top = 0;
        for (int w = 0; w < group / 64; ++w) top = s_top[w0 + w] > top ? s_top[w0 + w] : top;
        const QScale s = q_scale(top);
        if (mine) {
            if (at == 0) s_sa[row] = s.s;
            const int kp = g.ksteps * 64;
            for (int c = at * 4; c < kp; c += group * 4) {
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = c + j < q.k ? QElem<X>::load(x + c + j) : 0.f;
                *(unsigned*)(s_q + row * kp + c) = q_round4(f, s);
            }
        }
    }
    __syncthreads();
    const signed char* a = s_q + (r < q.rows ? r : (int)q.rows - 1) * (g.ksteps * 64) + kq;
    i32x4 acc = {0, 0, 0, 0};
    for (int s0 = wave; s0 < g.ksteps; s0 += FEW_WAVES * FEW_UNROLL) {
        if (s0 != wave) fetch(s0);
#pragma unroll
        for (int u = 0; u < FEW_UNROLL; ++u) {
            const int s = s0 + u * FEW_WAVES;
            if (s < g.ksteps) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u], *(const i32x4*)(a + s * 64), acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s_red[wave][r][(lane >> 4) * 4 + i] = acc[i];
    __syncthreads();
    if (tid < 256) {
        const int c = tid & 15, m = tid >> 4, n = n0 + c;
        if (m < g.m && n < g.n) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < FEW_WAVES; ++w) sum += s_red[w][m][c];
            float v = fmaf((float)sum * s_sa[m], g.sb[n], g.bias ? g.bias[n] : 0.f);
            if (g.relu && v < 0.f) v = 0.f;
            ((T*)g.y)[m * g.ldy + n] = YElem<T>::cvt(v);
        }
    }
}
template <typename X> static void linear_few(const I8Args& g, const QArgs& q, int dtype, hipStream_t st)
{
    int group = FEW_WAVES * 64;
    for (int m = 1; m < g.m; m *= 2) group /= 2;
    const dim3 grid((unsigned)cdiv(g.n, 16)), block(FEW_WAVES * 64);
    if (dtype == SAUNET_F32) hipLaunchKernelGGL((linear_int8_few_kernel<X, float>), grid, block, 0, st, g, q, group);
    else if (dtype == SAUNET_BF16) hipLaunchKernelGGL((linear_int8_few_kernel<X, u16>), grid, block, 0, st, g, q, group);
    else hipLaunchKernelGGL((linear_int8_few_kernel<X, _Float16>), grid, block, 0, st, g, q, group);
}

template <typename T> static int mm8_launch(const I8Args& g, hipStream_t st)
{
    // Little work: eight waves share the reduction of 16 channels x 32 (16) tokens.  Every such workgroup reads its operands for itself, so the tiles win from
    // some 512 workgroups on; us against the 64 x 64 tile, tokens x K x channels: 64 x 8075 x 1 7.6 / 28, 256 x 512 x 256 (128 workgroups) 2.8 / 4.5, 512 x 1024 x
    // 512 (512) 5.1 / 6.1, 64 x 4096 x 4096 (512) 13.7 / 15.5; 777 x 1001 x 515 (825) 7.8 / 7.4, 128 x 4096 x 4096 (1024) 24 / 16.  With 16 tokens or less the
    // weight is read once either way: to 16384 channels (1024 workgroups), 23.3 / 23.8.
    const long few = (g.m + 31) / 32 * ((g.n + 15) / 16);
    if (few <= (g.m <= 16 ? 1024 : 512)) {
        const dim3 grid((unsigned)cdiv(g.n, 16), g.m <= 16 ? 1 : (unsigned)((g.m + 31) / 32)), block(FEW_WAVES * 64);
        if (g.m <= 16) hipLaunchKernelGGL((matmul_int8_few_kernel<T, 1>), grid, block, 0, st, g);
        else hipLaunchKernelGGL((matmul_int8_few_kernel<T, 2>), grid, block, 0, st, g);
        SAUNET_CHECK_LAUNCH("matmul_int8_few");
        return SAUNET_OK;
    }
    const long t64 = ((g.m + 63) / 64) * ((g.n + 63) / 64);
    const long side = g.m < g.n ? g.m : g.n;
    if (side <= 64) return mm8_tiles<T, I8Core64>(g, st);
    if (t64 >= 192 * 16 && g.ksteps >= 8 && side > 192) return mm8_tiles<T, I8Core256>(g, st);
    if (t64 <= 384) return mm8_tiles<T, I8Core64>(g, st);
    if (t64 <= 768) return mm8_tiles<T, I8CoreTall>(g, st);
    return g.ksteps >= 64 ? mm8_tiles<T, I8Core128L>(g, st) : mm8_tiles<T, I8Core128>(g, st);
}

static int int8_check(const saunet_int8_desc* d, const char* who)
{
    if (!d || d->m < 0 || d->n < 1 || d->n > (1 << 30) || d->k < 1 || d->k > 131071) return set_error(SAUNET_BAD_SHAPE, "%s: bad sizes", who);
    const int64_t kp = (d->k + 63) / 64 * 64;
    if (d->ldb < kp || (d->ldb & 15) || d->ldb > (1 << 22) || d->ldy < d->n) return set_error(SAUNET_BAD_SHAPE, "%s: bad strides (%lld, %lld)", who, (long long)d->ldb, (long long)d->ldy);
    if (d->dtype != SAUNET_F32 && d->dtype != SAUNET_BF16 && d->dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "%s: dtype %d", who, d->dtype);
    if (d->m == 0) return SAUNET_OK;
    if (!d->b || !d->b_scale || !d->y) return set_error(SAUNET_BAD_SHAPE, "%s: missing memory", who);
    if ((uintptr_t)d->b & 15) return set_error(SAUNET_BAD_ALIGN, "%s: operands have to lie on a 16-byte border", who);
    return SAUNET_OK;
}
static I8Args int8_args(const saunet_int8_desc* d, const void* a, const float* sa, int64_t lda)
{
    const int size = d->dtype == SAUNET_F32 ? 4 : 2;
    return I8Args{(const char*)a, sa, lda, d->m, (const char*)d->b, d->b_scale, d->ldb, d->n, (d->k + 63) / 64, d->bias, d->relu, d->y, d->ldy,
                  !((uintptr_t)d->y & 15) && !(d->ldy * size & 15), 0};
}
static int int8_product(const saunet_int8_desc* d, const void* a, const float* sa, int64_t lda, hipStream_t st)
{
    const I8Args g = int8_args(d, a, sa, lda);
    if (d->dtype == SAUNET_F32) return mm8_launch<float>(g, st);
    if (d->dtype == SAUNET_BF16) return mm8_launch<u16>(g, st);
    return mm8_launch<_Float16>(g, st);
}

}  // namespace saunet

using namespace saunet;

extern "C" {

int saunet_quantize_rows(int dtype, const void* x, int64_t ldx, int64_t rows, int k, const float* scale, const float* shift, int relu, void* q, int64_t ldq, float* s, void* stream)
{
    if (rows < 0 || k < 1 || k > 131071 || ldx < k || ldq < k || (ldq & 63)) return set_error(SAUNET_BAD_SHAPE, "quantize_rows: %lld rows of %d (strides %lld -> %lld, whole 64-byte steps)", (long long)rows, k, (long long)ldx, (long long)ldq);
    if (dtype != SAUNET_F32 && dtype != SAUNET_BF16 && dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "quantize_rows: dtype %d", dtype);
    if (rows == 0) return SAUNET_OK;
    if (!x || !q || !s || (!scale) != (!shift)) return set_error(SAUNET_BAD_SHAPE, "quantize_rows: missing memory");
    if ((uintptr_t)q & 15) return set_error(SAUNET_BAD_ALIGN, "quantize_rows: q has to lie on a 16-byte border");
    const int size = dtype == SAUNET_F32 ? 4 : 2;
    hipStream_t st = (hipStream_t)stream;
    constexpr int64_t MOST = 1 << 23;                // rows a launch: up to 256 threads a row, and a launch has fewer than 2^32
    for (int64_t r0 = 0; r0 < rows; r0 += MOST) {
        const char* xr = (const char*)x + r0 * ldx * size;
        const QArgs a = {xr, ldx, rows - r0 < MOST ? rows - r0 : MOST, k, scale, shift, relu, (signed char*)q + r0 * ldq, ldq, s + r0,
                         !(((uintptr_t)xr | (uintptr_t)scale | (uintptr_t)shift) & 15) && !(ldx * size & 15)};
        if (scale || relu) dtype == SAUNET_F32 ? q_launch<float, true>(a, st) : dtype == SAUNET_BF16 ? q_launch<u16, true>(a, st) : q_launch<_Float16, true>(a, st);
        else dtype == SAUNET_F32 ? q_launch<float, false>(a, st) : dtype == SAUNET_BF16 ? q_launch<u16, false>(a, st) : q_launch<_Float16, false>(a, st);
        SAUNET_CHECK_LAUNCH("quantize_rows");
    }
    return SAUNET_OK;
}

int saunet_matmul_int8(const saunet_int8_desc* d, void* stream)
{
    const int rc = int8_check(d, "matmul_int8");
    if (rc) return rc;
    const int64_t kp = (d->k + 63) / 64 * 64;
    if (d->lda < kp || (d->lda & 15) || d->lda > (1 << 22)) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: bad stride %lld", (long long)d->lda);
    if (d->m == 0) return SAUNET_OK;
    if (!d->a || !d->a_scale) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: missing memory");
    if ((uintptr_t)d->a & 15) return set_error(SAUNET_BAD_ALIGN, "matmul_int8: operands have to lie on a 16-byte border");
    return int8_product(d, d->a, d->a_scale, d->lda, (hipStream_t)stream);
}

int saunet_linear_int8(const saunet_int8_desc* d, int x_dtype, const void* x, int64_t ldx, void* workspace, int64_t workspace_bytes, void* stream)
{
    const int rc = int8_check(d, "linear_int8");
    if (rc) return rc;
    if (x_dtype != SAUNET_F32 && x_dtype != SAUNET_BF16 && x_dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "linear_int8: dtype %d", x_dtype);
    if (ldx < d->k) return set_error(SAUNET_BAD_SHAPE, "linear_int8: bad stride %lld", (long long)ldx);
    if (d->m == 0) return SAUNET_OK;
    const int64_t kp = (d->k + 63) / 64 * 64;
    if (!x) return set_error(SAUNET_BAD_SHAPE, "linear_int8: missing memory");
    hipStream_t st = (hipStream_t)stream;
    if (d->m <= 8 && d->m * kp <= (d->m == 1 ? FEW_LDS : 4096)) {
        const I8Args g = int8_args(d, nullptr, nullptr, 0);
        const QArgs q = {x, ldx, d->m, d->k, nullptr, nullptr, 0, nullptr, 0, nullptr, 0};
        if (x_dtype == SAUNET_F32) linear_few<float>(g, q, d->dtype, st);
        else if (x_dtype == SAUNET_BF16) linear_few<u16>(g, q, d->dtype, st);
        else linear_few<_Float16>(g, q, d->dtype, st);
        SAUNET_CHECK_LAUNCH("linear_int8_few");
        return SAUNET_OK;
    }
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < d->m * (kp + 4)) return set_error(SAUNET_BAD_SHAPE, "linear_int8: the workspace has to hold %lld bytes on a 16-byte border", (long long)(d->m * (kp + 4)));
    float* s = (float*)((char*)workspace + d->m * kp);
    const int qc = saunet_quantize_rows(x_dtype, x, ldx, d->m, d->k, nullptr, nullptr, 0, workspace, kp, s, stream);
    return qc ? qc : int8_product(d, workspace, s, kp, st);
}

}  // extern "C"
