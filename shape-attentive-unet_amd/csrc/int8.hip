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

struct QArgs { const void* x; long ldx; long rows; int k; const float* scale; const float* shift; int relu; signed char* q; long ldq; float* s; int vec; };

// G lanes a row, NV vectors a lane kept in registers (k <= G * NV * V, 16-byte aligned rows); NV == 0: any k and alignment, the row is read twice
template <typename T, int G, int NV> __global__ __launch_bounds__(256) void quantize_rows_kernel(QArgs a)
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
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (c + V <= a.k) v = *(const u32x4*)(x + c);
            QElem<T>::unpack(v, f[i]);
            if (c < a.k && c + V > a.k) for (int j = 0; j < V; ++j) f[i][j] = c + j < a.k ? QElem<T>::load(x + c + j) : 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (c + j < a.k) f[i][j] = pro(f[i][j], c + j);
                const unsigned b = __float_as_uint(f[i][j]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) { const unsigned b = __shfl_xor(top, o, G); top = b > top ? b : top; }
        const QScale s = q_scale(top);
        if (lane == 0) a.s[row] = s.s;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            if (c >= a.ldq) continue;
            unsigned w[2] = {0u, 0u};
#pragma unroll
            for (int j = 0; j < V; ++j) w[j >> 2] |= ((unsigned)q_round(f[i][j], s) & 255u) << ((j & 3) * 8);
            if (V == 8) *(u32x2*)(q + c) = u32x2{w[0], w[1]};
            else *(unsigned*)(q + c) = w[0];
        }
        for (int c = (NV * G + lane) * V; c < a.ldq; c += G * V) {       // padding beyond the registers' reach
            if (V == 8) *(u32x2*)(q + c) = u32x2{0u, 0u};
            else *(unsigned*)(q + c) = 0u;
        }
    } else {
        for (int c = lane; c < a.k; c += G) { const unsigned b = __float_as_uint(pro(QElem<T>::load(x + c), c)) & 0x7fffffffu; top = b > top ? b : top; }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) { const unsigned b = __shfl_xor(top, o, G); top = b > top ? b : top; }
        const QScale s = q_scale(top);
        if (lane == 0) a.s[row] = s.s;
        for (int c = lane * 4; c < a.ldq; c += G * 4) {
            unsigned w = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) if (c + j < a.k) w |= ((unsigned)q_round(pro(QElem<T>::load(x + c + j), c + j), s) & 255u) << (j * 8);
            *(unsigned*)(q + c) = w;
        }
    }
}

template <typename T> static void q_launch(const QArgs& a, hipStream_t st)
{
    constexpr int V = QElem<T>::V;
#define Q_GO(G, NV) hipLaunchKernelGGL((quantize_rows_kernel<T, G, NV>), dim3((unsigned)((a.rows + 256 / G - 1) / (256 / G))), dim3(256), 0, st, a)
    if (!a.vec) Q_GO(64, 0);
    else if (a.k <= 16 * V) Q_GO(16, 1);
    else if (a.k <= 32 * V) Q_GO(16, 2);
    else if (a.k <= 64 * V) Q_GO(64, 1);
    else if (a.k <= 128 * V) Q_GO(64, 2);
    else if (a.k <= 256 * V) Q_GO(64, 4);
    else if (a.k <= 512 * V) Q_GO(64, 8);
    else Q_GO(64, 0);
#undef Q_GO
}

// ---- the product ------------------------------------------------------------------------------------------------------------------
struct I8Args { const char* a; const float* sa; long lda; long m; const char* b; const float* sb; long ldb; int n; int ksteps; const float* bias; int relu; void* y; long ldy; int vec; int tn; };

template <typename T> struct YElem;
template <> struct YElem<float> { static __device__ __forceinline__ float cvt(float v) { return v; } };
template <> struct YElem<u16> { static __device__ __forceinline__ u16 cvt(float v) { return __builtin_bit_cast(u16, (__bf16)v); } };
template <> struct YElem<_Float16> { static __device__ __forceinline__ _Float16 cvt(float v) { return (_Float16)v; } };

// Operand A of the MFMA is the WEIGHT tile (BM channels), operand B the token tile (BN tokens): a lane then holds four consecutive channels of one token.
// The wave's 32 tokens x (BM / WGM) channels go through LDS so that the stores are whole rows of the tile.
template <typename T, class Core> __global__ __launch_bounds__(Core::NT) void matmul_int8_kernel(I8Args g)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int tn = g.tn, id = blockIdx.x;                       // channel tiles run fastest: the workgroups beside each other share the token tile
    const long m0 = (long)(id / tn) * Core::BN;
    const int n0 = (id % tn) * Core::BM;
    typename Core::Acc acc[Core::TM][Core::TN] = {};
    const long ml = g.m - m0;
    Core::run(g.b + (long)n0 * g.ldb, (unsigned)g.ldb, g.n - n0, g.a + m0 * g.lda, (unsigned)g.lda, ml < Core::BN ? (int)ml : Core::BN, g.ksteps, smem, acc);
    __syncthreads();
    constexpr int CH = Core::BM / Core::WGM, PITCH = CH * (int)sizeof(T) + 16;          // one wave: 32 tokens of CH channels
    static_assert(Core::NW * 32 * PITCH <= 160 * 1024, "the wave's rows fit");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / Core::WGN, wn = wave % Core::WGN, half = lane >> 5, tok = lane & 31;
    unsigned char* buf = smem + wave * 32 * PITCH;
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
                T o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = nw + c + r < g.n ? nw + c + r : g.n - 1;
                    float v = (float)acc[ti][tj][q * 4 + r] * sa * g.sb[n];
                    if (g.bias) v += g.bias[n];
                    if (g.relu && v < 0.f) v = 0.f;
                    o[r] = YElem<T>::cvt(v);
                }
                if (sizeof(T) == 4) *(u32x4*)(buf + tok * PITCH + c * sizeof(T)) = *(const u32x4*)o;
                else *(u32x2*)(buf + tok * PITCH + c * sizeof(T)) = *(const u32x2*)o;
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

typedef NtCore<NtI8, 128, 128, 2, 2, 4> I8Core128;

template <typename T> static int mm8_launch(I8Args g, hipStream_t st)
{
    typedef I8Core128 Core;
    constexpr int EPI = Core::NW * 32 * (Core::BM / Core::WGM * (int)sizeof(T) + 16), LDS = Core::LDS > EPI ? Core::LDS : EPI;
    static DeviceOnce once;
    if (once.first()) (void)hipFuncSetAttribute((const void*)matmul_int8_kernel<T, Core>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    g.tn = cdiv(g.n, Core::BM);
    const long tiles = (g.m + Core::BN - 1) / Core::BN * g.tn;
    if (tiles > 0x7fffffff) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: %ld tiles", tiles);
    hipLaunchKernelGGL((matmul_int8_kernel<T, Core>), dim3((unsigned)tiles), dim3(Core::NT), LDS, st, g);
    SAUNET_CHECK_LAUNCH("matmul_int8");
    return SAUNET_OK;
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
    if (rows > 0x7fffffffL * 4) return set_error(SAUNET_BAD_SHAPE, "quantize_rows: %lld rows", (long long)rows);
    const int size = dtype == SAUNET_F32 ? 4 : 2;
    QArgs a = {x, ldx, rows, k, scale, shift, relu, (signed char*)q, ldq, s, !((uintptr_t)x & 15) && !(ldx * size & 15)};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SAUNET_F32) q_launch<float>(a, st);
    else if (dtype == SAUNET_BF16) q_launch<u16>(a, st);
    else q_launch<_Float16>(a, st);
    SAUNET_CHECK_LAUNCH("quantize_rows");
    return SAUNET_OK;
}

int saunet_matmul_int8(const saunet_int8_desc* d, void* stream)
{
    if (!d || d->m < 0 || d->n < 1 || d->k < 1 || d->k > 131071) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: bad sizes");
    const int64_t kp = (d->k + 63) / 64 * 64;
    if (d->lda < kp || d->ldb < kp || (d->lda & 15) || (d->ldb & 15) || d->lda > (1 << 22) || d->ldb > (1 << 22) || d->ldy < d->n) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: bad strides (%lld, %lld, %lld)", (long long)d->lda, (long long)d->ldb, (long long)d->ldy);
    if (d->dtype != SAUNET_F32 && d->dtype != SAUNET_BF16 && d->dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "matmul_int8: dtype %d", d->dtype);
    if (d->m == 0) return SAUNET_OK;
    if (!d->a || !d->b || !d->a_scale || !d->b_scale || !d->y) return set_error(SAUNET_BAD_SHAPE, "matmul_int8: missing memory");
    if (((uintptr_t)d->a | (uintptr_t)d->b) & 15) return set_error(SAUNET_BAD_ALIGN, "matmul_int8: operands have to lie on a 16-byte border");
    const int size = d->dtype == SAUNET_F32 ? 4 : 2;
    I8Args g = {(const char*)d->a, d->a_scale, d->lda, d->m, (const char*)d->b, d->b_scale, d->ldb, d->n, (int)(kp / 64), d->bias, d->relu, d->y, d->ldy,
                !((uintptr_t)d->y & 15) && !(d->ldy * size & 15), 0};
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == SAUNET_F32) return mm8_launch<float>(g, st);
    if (d->dtype == SAUNET_BF16) return mm8_launch<u16>(g, st);
    return mm8_launch<_Float16>(g, st);
}

}  // extern "C"
