// Newton-Schulz orthogonalisation of a list of matrices and the Muon step around it.
//
//   X0 = G / max(|G|_F, eps);   S = X X^T,  X <- (a I + b S + c S^2) X,  `steps` times          (rows <= columns; the transpose otherwise)
//
// One call takes any number of matrices of any shapes: every launch below covers one phase of ALL of them, a workgroup finds its matrix in a
// table of tile prefixes.  The whole chain is some twenty launches whatever the list is.
//
// Composition.  S_k+1 = P_k S_k P_k with P_k = a I + b S_k + c S_k^2, and all of them commute, so up to three steps run on the m x m matrices alone
// (S and the product Q = P_2 P_1 P_0) before X is touched: 6 m^2 n + 14 m^3 operations for five steps (3 + 2) against 5 (3 m^2 n + m^3).  Equal for a
// square, 2.4x less at n = 27 m.  An error of S grows by a^2 = 12 with every step it is carried through, so S is formed anew from X after three:
// composing all five loses four digits, composing three + two none (1.0e-6 against 0.5e-6 of |X|; the same chain in float32: 2e-6 .. 1e-5).
// What is composed is (P_2 P_1 P_0 - a^3 I): up to 41 in size where s is near 1, for a result near 1.  Since the s^2 add up to 1, that costs
// 41 / sqrt(m) roundings of the result's norm -- nothing from m = 32 on, two digits at m = 1, so a list with a shorter matrix goes step by step.
//
// Number format.  Every matrix between the first and the last pass is a pair of float16 planes, x = hi + lo to 2^-24 (nt_tiles.h: 128-byte blocks of 32
// elements), scaled by a power of two that the host derives from the singular values' range.  A product is then three float16 MFMAs with float32
// accumulation, at a sixth of the cost of the float32 MFMA and with no more error.  Products of symmetric matrices compute the lower tiles only and
// write both halves.  X and X^T are both kept: each is the operand with the contiguous reduction index in one of the two rectangular products.
#include "nt_tiles.h"

namespace saunet {

struct NsItem {            // 72 bytes: one matrix, as the host lays it out
    const void* src; void* dst; float* buf; char* ws;
    int ld_src, ld_dst, rows, cols, splits;
    int p_norm, p_pack, p_sym, p_gram, p_app;       // index of the matrix's first workgroup in the launches of each kind
};
constexpr int NS_CHUNK = 52;
struct NsItems { NsItem it[NS_CHUNK]; };
constexpr int NS_TILE = 128, NS_NORM = 8192;        // elements a workgroup of the norm pass takes

enum { NS_A = 0, NS_P, NS_R, NS_Q0, NS_Q1, NS_NSYM };
struct NsView {
    int m, n, mp, np, tall;
    char *x, *xt[2], *sym[NS_NSYM]; float* part;
    __host__ __device__ static long bytes(int rows, int cols, int splits)
    {
        const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows, mp = (m + 31) / 32 * 32, np = (n + 31) / 32 * 32, t = (m + NS_TILE - 1) / NS_TILE;
        return 3 * mp * np * 4 + NS_NSYM * mp * mp * 4 + (splits > 1 ? (long)splits * (t * (t + 1) / 2) * NS_TILE * NS_TILE * 4 : 0);
    }
    __device__ explicit NsView(const NsItem& it)
    {
        tall = it.rows > it.cols;
        m = tall ? it.cols : it.rows; n = tall ? it.rows : it.cols;
        mp = (m + 31) / 32 * 32; np = (n + 31) / 32 * 32;
        const long bx = (long)mp * np * 4, bs = (long)mp * mp * 4;
        char* p = it.ws;
        x = p; p += bx; xt[0] = p; p += bx; xt[1] = p; p += bx;
        for (int i = 0; i < NS_NSYM; ++i) { sym[i] = p; p += bs; }
        part = (float*)p;
    }
};

// the matrix whose workgroups include `id` of the launches of this kind; two rounds of one load a lane (count <= 4096)
template <int NsItem::*P> __device__ __forceinline__ int ns_find(const NsItem* __restrict__ tab, int count, int id)
{
    const int lane = threadIdx.x & 63, step = (count + 63) >> 6;
    int base = 0;
    if (step > 1) {
        const int i = lane * step;
        base = (__popcll(__ballot(i < count && tab[i].*P <= id)) - 1) * step;
    }
    const int i = base + lane;
    return __builtin_amdgcn_readfirstlane(base + __popcll(__ballot(lane < step * (step > 1) + 64 * (step <= 1) && i < count && tab[i].*P <= id)) - 1);
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
template <typename T, bool MUON> __global__ __launch_bounds__(256) void ns_norm_kernel(const NsItem* __restrict__ tab, int count, const float* __restrict__ hyper, double* __restrict__ part)
{
    __shared__ double s_sum[4];
    const int id = blockIdx.x;
    const NsItem it = tab[ns_find<&NsItem::p_norm>(tab, count, id)];
    const long total = (long)it.rows * it.cols, e0 = (long)(id - it.p_norm) * NS_NORM;
    float h[5] = {0.f, 0.f, 0.f, 0.f, 1.f};
    if (MUON) for (int i = 0; i < 5; ++i) h[i] = hyper[i];
    double sum = 0.0;
    auto one = [&](long e, float g) {
        float u = g;
        if (MUON) { const float b = ns_momentum(g, it.buf[e], h); it.buf[e] = b; u = ns_update(g, b, h); }
        sum += (double)u * (double)u;
    };
    if (it.ld_src == it.cols) {
        for (int k = threadIdx.x; k < NS_NORM; k += 256) { const long e = e0 + k; if (e < total) one(e, ns_load((const T*)it.src + e)); }
    } else {
        for (int k = threadIdx.x; k < NS_NORM; k += 256) {
            const long e = e0 + k;
            if (e < total) { const long r = e / it.cols; one(e, ns_load((const T*)it.src + r * it.ld_src + (e - r * it.cols))); }
        }
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[id] = ((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3];
}

// ---- X0 and X0^T as scaled float16 pairs: a workgroup takes 64 x 64 elements --------------------------------------------------------
template <typename T, bool MUON> __global__ __launch_bounds__(256) void ns_pack_kernel(const NsItem* __restrict__ tab, int count, const float* __restrict__ hyper, const double* __restrict__ part, float eps, float sx)
{
    __shared__ float s_t[64][65];
    __shared__ double s_sum[4];
    const int tid = threadIdx.x, id = blockIdx.x;
    const NsItem it = tab[ns_find<&NsItem::p_pack>(tab, count, id)];
    const NsView v(it);
    const int nblk = (int)(((long)it.rows * it.cols + NS_NORM - 1) / NS_NORM);
    double sum = 0.0;
    for (int i = tid; i < nblk; i += 256) sum += part[it.p_norm + i];
    sum = wave_sum(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    const double norm = sqrt(((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3]);
    const double inv = (double)sx / (norm <= (double)eps ? (double)eps : norm);      // a NaN norm stays NaN
    float h[5] = {0.f, 0.f, 0.f, 0.f, 1.f};
    if (MUON) for (int i = 0; i < 5; ++i) h[i] = hyper[i];
    // tiles in the caller's orientation: r along its rows, c along its columns
    const int rp = v.tall ? v.np : v.mp, cp = v.tall ? v.mp : v.np, tc = (cp + 63) / 64, t = id - it.p_pack;
    const int r0 = t / tc * 64, c0 = t % tc * 64;
    for (int k = tid; k < 64 * 64; k += 256) {
        const int r = r0 + (k >> 6), c = c0 + (k & 63);
        float u = 0.f;
        if (r < it.rows && c < it.cols) {
            u = ns_load((const T*)it.src + (long)r * it.ld_src + c);
            if (MUON) u = ns_update(u, it.buf[(long)r * it.cols + c], h);
            u = (float)((double)u * inv);
        }
        s_t[k >> 6][k & 63] = u;
    }
    __syncthreads();
    // 8 consecutive elements a thread: 16 bytes of high and of low parts; along[] runs along the caller's rows, across[] along its columns
    char* along = v.tall ? v.xt[0] : v.x;
    char* across = v.tall ? v.x : v.xt[0];
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
typedef NtCore<NtF16Pair, NS_TILE, NS_TILE, 2, 2, 2> NsCore;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;

struct NsTile { int i0, j0; };          // the wave's corner in C
// calls f(i, j, value[4]) for the 4 consecutive rows i .. i + 3 and the column j of every accumulator quad inside [0, mlim) x [0, nlim) (multiples of 32)
template <typename F> __device__ __forceinline__ void ns_for_quads(f32x16 (&acc)[NsCore::TM][NsCore::TN], int i0, int j0, int mlim, int nlim, F f)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int ti = 0; ti < NsCore::TM; ++ti)
#pragma unroll
        for (int tj = 0; tj < NsCore::TN; ++tj) {
            if (i0 + ti * 32 >= mlim || j0 + tj * 32 >= nlim) continue;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float q[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) q[r] = acc[ti][tj][g * 4 + r];
                f(i0 + ti * 32 + g * 8 + (lane >> 5) * 4, j0 + tj * 32 + (lane & 31), q);
            }
        }
}
// four consecutive elements (row j, columns i .. i + 3) of a pair matrix with lda bytes a row
__device__ __forceinline__ void ns_read4(const char* p, long ldb, int j, int i, float (&v)[4])
{
    const char* s = p + (long)j * ldb + (i >> 5) * 128 + (i & 31) * 2;
    const f16x4_t h = *(const f16x4_t*)s, l = *(const f16x4_t*)(s + 64);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (float)h[r] + (float)l[r];
}
// value (i .. i + 3, j) to row j of dt and to the rows i .. i + 3 of d
__device__ __forceinline__ void ns_write4(char* dt, long ldt, char* d, long ldd, int i, int j, const float (&v)[4])
{
    f16x4_t h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) { const Pair s = ns_split(v[r]); h[r] = s.h; l[r] = s.l; }
    char* p = dt + (long)j * ldt + (i >> 5) * 128 + (i & 31) * 2;
    *(f16x4_t*)p = h; *(f16x4_t*)(p + 64) = l;
    char* q = d + (long)i * ldd + (j >> 5) * 128 + (j & 31) * 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) { *(_Float16*)(q + r * ldd) = h[r]; *(_Float16*)(q + r * ldd + 64) = l[r]; }
}
// the same into a symmetric matrix: of a tile on the diagonal the upper part is dropped, so that the stored matrix is symmetric to the last bit.  An
// antisymmetric rounding error would not shrink with a I + P as the error of S does: it grew six-fold a product (2e-5 of |X| after five steps).
__device__ __forceinline__ void ns_write4_sym(char* d, long ld, bool diag, int i, int j, const float (&v)[4])
{
    if (!diag || i >= j) { ns_write4(d, ld, d, ld, i, j, v); return; }
    if (i + 3 < j) return;
#pragma unroll
    for (int r = 1; r < 4; ++r) {
        if (i + r < j) continue;
        const Pair s = ns_split(v[r]);
        char* p = d + (long)j * ld + ((i + r) >> 5) * 128 + ((i + r) & 31) * 2;
        char* q = d + (long)(i + r) * ld + (j >> 5) * 128 + (j & 31) * 2;
        *(_Float16*)p = s.h; *(_Float16*)(p + 64) = s.l;
        *(_Float16*)q = s.h; *(_Float16*)(q + 64) = s.l;
    }
}
// tile t of the lower triangle, row by row: (ti, tj), tj <= ti
__device__ __forceinline__ void ns_lower(int t, int& ti, int& tj)
{
    ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    while (ti * (ti + 1) / 2 > t) --ti;
    tj = t - ti * (ti + 1) / 2;
}

// S = X X^T: lower tiles, the columns in it.splits parts.  One part: straight to S.  More: float32 partials in accumulator order for ns_gram_finish.
__global__ __launch_bounds__(256, 2) void ns_gram_kernel(const NsItem* __restrict__ tab, int count, float alpha)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int id = blockIdx.x;
    const NsItem it = tab[ns_find<&NsItem::p_gram>(tab, count, id)];
    const NsView v(it);
    const int t = (id - it.p_gram) / it.splits, sp = (id - it.p_gram) % it.splits;
    int ti, tj;
    ns_lower(t, ti, tj);
    const int steps = v.np / 32, k0 = (int)((long)steps * sp / it.splits), k1 = (int)((long)steps * (sp + 1) / it.splits);
    f32x16 acc[NsCore::TM][NsCore::TN] = {};
    const long ld = (long)v.np * 4;
    NsCore::run(v.x + ti * NS_TILE * ld + k0 * 128, (unsigned)ld, v.mp - ti * NS_TILE, v.x + tj * NS_TILE * ld + k0 * 128, (unsigned)ld, v.mp - tj * NS_TILE, k1 - k0, smem, acc);
    const int wave = threadIdx.x >> 6, i0 = ti * NS_TILE + (wave >> 1) * 64, j0 = tj * NS_TILE + (wave & 1) * 64;
    if (it.splits > 1) {
        float* p = v.part + ((long)t * it.splits + sp) * NS_TILE * NS_TILE + threadIdx.x * 4;
#pragma unroll
        for (int b = 0; b < 16; ++b) *(f32x4*)(p + b * 1024) = f32x4{acc[b >> 3][(b >> 2) & 1][(b & 3) * 4], acc[b >> 3][(b >> 2) & 1][(b & 3) * 4 + 1], acc[b >> 3][(b >> 2) & 1][(b & 3) * 4 + 2], acc[b >> 3][(b >> 2) & 1][(b & 3) * 4 + 3]};
        return;
    }
    char* s = v.sym[NS_A];
    ns_for_quads(acc, i0, j0, v.mp, v.mp, [&](int i, int j, const float (&q)[4]) {
        const float w[4] = {alpha * q[0], alpha * q[1], alpha * q[2], alpha * q[3]};
        ns_write4_sym(s, v.mp * 4L, ti == tj, i, j, w);
    });
}
__global__ __launch_bounds__(256) void ns_gram_finish_kernel(const NsItem* __restrict__ tab, int count, float alpha)
{
    const int id = blockIdx.x;
    const NsItem it = tab[ns_find<&NsItem::p_sym>(tab, count, id)];
    if (it.splits < 2) return;
    const NsView v(it);
    const int t = id - it.p_sym;
    int ti, tj;
    ns_lower(t, ti, tj);
    f32x16 acc[NsCore::TM][NsCore::TN] = {};
    const float* p = v.part + (long)t * it.splits * NS_TILE * NS_TILE + threadIdx.x * 4;
    for (int sp = 0; sp < it.splits; ++sp, p += NS_TILE * NS_TILE)
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const f32x4 w = *(const f32x4*)(p + b * 1024);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[b >> 3][(b >> 2) & 1][(b & 3) * 4 + r] += w[r];
        }
    const int wave = threadIdx.x >> 6, i0 = ti * NS_TILE + (wave >> 1) * 64, j0 = tj * NS_TILE + (wave & 1) * 64;
    char* s = v.sym[NS_A];
    ns_for_quads(acc, i0, j0, v.mp, v.mp, [&](int i, int j, const float (&q)[4]) {
        const float w[4] = {alpha * q[0], alpha * q[1], alpha * q[2], alpha * q[3]};
        ns_write4_sym(s, v.mp * 4L, ti == tj, i, j, w);
    });
}

// D = alpha A B + beta E + gamma F over symmetric matrices that commute (so D is symmetric): lower tiles, both halves written.  blockIdx.y picks the
// product: the two of one phase are independent.
struct NsProd { int a, b, e, f, d; float alpha, beta, gamma; };
struct NsProds { NsProd p[2]; };
__global__ __launch_bounds__(256, 2) void ns_sym_kernel(const NsItem* __restrict__ tab, int count, NsProds pr)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int id = blockIdx.x;
    const NsProd p = pr.p[blockIdx.y];
    const NsItem it = tab[ns_find<&NsItem::p_sym>(tab, count, id)];
    const NsView v(it);
    int ti, tj;
    ns_lower(id - it.p_sym, ti, tj);
    f32x16 acc[NsCore::TM][NsCore::TN] = {};
    const long ld = (long)v.mp * 4;
    NsCore::run(v.sym[p.a] + ti * NS_TILE * ld, (unsigned)ld, v.mp - ti * NS_TILE, v.sym[p.b] + tj * NS_TILE * ld, (unsigned)ld, v.mp - tj * NS_TILE, v.mp / 32, smem, acc);
    const int wave = threadIdx.x >> 6, i0 = ti * NS_TILE + (wave >> 1) * 64, j0 = tj * NS_TILE + (wave & 1) * 64;
    const char* e = v.sym[p.e];
    const char* f = p.f < 0 ? nullptr : v.sym[p.f];
    char* d = v.sym[p.d];
    ns_for_quads(acc, i0, j0, v.mp, v.mp, [&](int i, int j, const float (&q)[4]) {
        float w[4], x[4];
        ns_read4(e, ld, j, i, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fmaf(p.alpha, q[r], p.beta * x[r]);
        if (f) {
            ns_read4(f, ld, j, i, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = fmaf(p.gamma, x[r], w[r]);
        }
        ns_write4_sym(d, ld, ti == tj, i, j, w);
    });
}

// X <- alpha Q X + beta X.  MODE 0: back to X and the other X^T; 1: to the caller's matrix; 2: the Muon update of the caller's parameter
template <typename T, int MODE> __global__ __launch_bounds__(256, 2) void ns_apply_kernel(const NsItem* __restrict__ tab, int count, int q, int xt, float alpha, float beta, const float* __restrict__ hyper, int adjust)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int id = blockIdx.x;
    const NsItem it = tab[ns_find<&NsItem::p_app>(tab, count, id)];
    const NsView v(it);
    const int tm = (v.mp + NS_TILE - 1) / NS_TILE, t = id - it.p_app, ti = t % tm, tj = t / tm;
    f32x16 acc[NsCore::TM][NsCore::TN] = {};
    const long ld = (long)v.mp * 4;
    NsCore::run(v.sym[q] + ti * NS_TILE * ld, (unsigned)ld, v.mp - ti * NS_TILE, v.xt[xt] + tj * NS_TILE * ld, (unsigned)ld, v.np - tj * NS_TILE, v.mp / 32, smem, acc);
    const int wave = threadIdx.x >> 6, i0 = ti * NS_TILE + (wave >> 1) * 64, j0 = tj * NS_TILE + (wave & 1) * 64;
    const char* x = v.xt[xt];
    float keep = 0.f, rate = 0.f;
    if (MODE == 2) {
        const float lr = hyper[0], big = (float)(it.rows > it.cols ? it.rows : it.cols);
        keep = 1.f - lr * hyper[2];
        rate = lr * (adjust ? 0.2f * sqrtf(big) : it.rows > it.cols ? sqrtf((float)it.rows / (float)it.cols) : 1.f);
    }
    ns_for_quads(acc, i0, j0, v.mp, v.np, [&](int i, int j, const float (&a)[4]) {
        float w[4], o[4];
        ns_read4(x, ld, j, i, o);
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fmaf(alpha, a[r], beta * o[r]);
        if (MODE == 0) { ns_write4(v.xt[xt ^ 1], ld, v.x, v.np * 4L, i, j, w); return; }
        if (j >= v.n) return;
        T* d = (T*)it.dst + (v.tall ? (long)j * it.ld_dst + i : (long)i * it.ld_dst + j);
        const long st = v.tall ? 1 : it.ld_dst;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (i + r >= v.m) break;
            if (MODE == 1) ns_store(d + r * st, w[r]);
            else d[r * st] = (T)fmaf(-rate, w[r], keep * (float)d[r * st]);
        }
    });
}

// ---- host side --------------------------------------------------------------------------------------------------------------------------------
struct NsPlan { long norm, pack, sym, gram, app, tab_bytes, part_bytes, bytes, shortest; bool split; };

static int ns_check(const saunet_ns_desc* d, const char* who)
{
    if (!d || !d->item || d->count < 1 || d->count > 4096) return set_error(SAUNET_BAD_SHAPE, "%s: 1 to 4096 matrices, not %d", who, d ? d->count : 0);
    if (d->dtype != SAUNET_F32 && d->dtype != SAUNET_BF16 && d->dtype != SAUNET_F16) return set_error(SAUNET_BAD_DTYPE, "%s: dtype %d", who, d->dtype);
    if (d->steps < 1 || d->steps > 32) return set_error(SAUNET_BAD_SHAPE, "%s: 1 to 32 steps, not %d", who, d->steps);
    if (!(d->eps > 0.f)) return set_error(SAUNET_BAD_SHAPE, "%s: eps has to be positive", who);
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        if (t.rows < 1 || t.cols < 1 || t.rows > (1 << 20) || t.cols > (1 << 20) || (t.rows > 32768 && t.cols > 32768))
            return set_error(SAUNET_BAD_SHAPE, "%s: matrix %d is %d x %d (sides up to 2^20, the shorter up to 32768)", who, i, t.rows, t.cols);
        if (t.ld_src < t.cols || t.ld_dst < t.cols || t.ld_src > 0x7fffffff || t.ld_dst > 0x7fffffff) return set_error(SAUNET_BAD_SHAPE, "%s: matrix %d has a bad row stride", who, i);
    }
    return SAUNET_OK;
}

// tile counts, prefixes (into `out` when given) and the workspace: table | norm partials | matrices
static int ns_plan(const saunet_ns_desc* d, NsPlan& p, NsItem* out, char* ws)
{
    p = NsPlan();
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        const long m = t.rows < t.cols ? t.rows : t.cols, n = t.rows < t.cols ? t.cols : t.rows;
        const long tm = (m + NS_TILE - 1) / NS_TILE;
        p.sym += tm * (tm + 1) / 2;
        p.norm += (m * n + NS_NORM - 1) / NS_NORM;
        if (i == 0 || m < p.shortest) p.shortest = m;
    }
    p.tab_bytes = ((long)sizeof(NsItem) * d->count + 255) / 256 * 256;
    p.part_bytes = (p.norm * 8 + 255) / 256 * 256;
    // a Gram tile walks the whole long side: it is split until the launch has about 1024 workgroups, each part 512 columns at least
    const long want = p.sym < 1024 ? 1024 / p.sym : 1;
    long at = p.tab_bytes + p.part_bytes;
    long norm = 0, sym = 0;
    for (int i = 0; i < d->count; ++i) {
        const saunet_ns_item& t = d->item[i];
        const long m = t.rows < t.cols ? t.rows : t.cols, n = t.rows < t.cols ? t.cols : t.rows;
        const long tm = (m + NS_TILE - 1) / NS_TILE, tn = (n + NS_TILE - 1) / NS_TILE, mp = (m + 31) / 32 * 32, np = (n + 31) / 32 * 32;
        long splits = np / 512 < want ? np / 512 : want;
        if (splits < 1) splits = 1;
        if (splits > 1) p.split = true;
        if (out) {
            NsItem& o = out[i];
            o.src = t.src; o.dst = t.dst; o.buf = (float*)t.buf; o.ws = ws + at;
            o.ld_src = (int)t.ld_src; o.ld_dst = (int)t.ld_dst; o.rows = t.rows; o.cols = t.cols; o.splits = (int)splits;
            o.p_norm = (int)norm; o.p_pack = (int)p.pack; o.p_sym = (int)sym; o.p_gram = (int)p.gram; o.p_app = (int)p.app;
        }
        norm += (m * n + NS_NORM - 1) / NS_NORM;
        sym += tm * (tm + 1) / 2;
        p.pack += ((mp + 63) / 64) * ((np + 63) / 64);
        p.gram += tm * (tm + 1) / 2 * splits;
        p.app += tm * tn;
        at += (NsView::bytes(t.rows, t.cols, (int)splits) + 255) / 256 * 256;
    }
    p.bytes = at;
    if (p.norm > 0x7fffffff || p.pack > 0x7fffffff || p.gram > 0x7fffffff || p.app > 0x7fffffff || p.sym > 0x7fffffff) return set_error(SAUNET_BAD_SHAPE, "newton_schulz: the list is too large for one call");
    return SAUNET_OK;
}

// Largest magnitude that a matrix with eigenvalue f(s), s in [0, 1] the first singular values, can hold: its power-of-two scale leaves a factor of two
// below the largest float16.  The grid is even in s^(1/4): small singular values grow fastest.
constexpr int NS_GRID = 2048;
static float ns_scale(const double* v)
{
    double top = 1e-3;
    for (int i = 0; i <= NS_GRID; ++i) { const double a = v[i] < 0 ? -v[i] : v[i]; if (!(a <= 1e30)) return 0.f; if (a > top) top = a; }
    double s = 32768.0;
    while (s * top > 32768.0) s *= 0.5;
    while (s * top * 2.0 <= 32768.0 && s < 16384.0 * 64) s *= 2.0;
    return (float)s;
}

template <typename T, bool MUON> static int ns_run(const saunet_ns_desc* d, const float* hyper, void* workspace, int64_t workspace_bytes, hipStream_t st, const char* who)
{
    NsPlan p;
    int rc = ns_plan(d, p, nullptr, nullptr);
    if (rc) return rc;
    if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255)) return set_error(SAUNET_BAD_SHAPE, "%s: the workspace has to hold %ld bytes on a 256-byte border", who, p.bytes);
    // the scalar iteration on a grid of singular values: ranges of every intermediate matrix, from which its scale follows
    static thread_local double x[NS_GRID + 1], S[NS_GRID + 1], P[NS_GRID + 1], Q[NS_GRID + 1], R[NS_GRID + 1];
    static thread_local NsItem items[4096];
    char* ws = (char*)workspace;
    rc = ns_plan(d, p, items, ws);
    if (rc) return rc;
    NsItem* tab = (NsItem*)ws;
    double* part = (double*)(ws + p.tab_bytes);
    const int n = d->count;
    const double a = d->a, b = d->b, c = d->c;
    // first check that every scale exists, launching nothing; then the same walk with launches
    for (int go = 0; go < 2; ++go) {
        for (int i = 0; i <= NS_GRID; ++i) { const double u = (double)i / NS_GRID; x[i] = u * u * u * u * (1.0 + 1e-6); }
        float sx = ns_scale(x);
        if (go) {
            for (int i = 0; i < n; i += NS_CHUNK) {
                NsItems ch;
                const int k = n - i < NS_CHUNK ? n - i : NS_CHUNK;
                memcpy(ch.it, items + i, sizeof(NsItem) * k);
                hipLaunchKernelGGL(ns_setup_kernel, dim3(1), dim3(64), 0, st, ch, k, tab + i);
            }
            hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)p.norm), dim3(256), 0, st, tab, n, hyper, part);
            hipLaunchKernelGGL((ns_pack_kernel<T, MUON>), dim3((unsigned)p.pack), dim3(256), 0, st, tab, n, hyper, part, d->eps, sx);
            SAUNET_CHECK_LAUNCH("ns_pack");
        }
        int xt = 0;
        for (int done = 0; done < d->steps;) {
            // three steps at a time on the Gram matrix while a^2 each keeps its rounding error below 2^8 of itself, else one
            const int left = d->steps - done;
            int nb = a * a <= 16.0 && p.shortest >= 32 ? (left == 4 ? 2 : left < 3 ? left : 3) : 1;
            for (int i = 0; i <= NS_GRID; ++i) S[i] = x[i] * x[i];
            float sa = ns_scale(S), sp = 0, sq = 0;
            if (sa == 0.f || sx == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
            if (go) {
                const float alpha = sa / (sx * sx);
                hipLaunchKernelGGL(ns_gram_kernel, dim3((unsigned)p.gram), dim3(256), NsCore::LDS, st, tab, n, alpha);
                SAUNET_CHECK_LAUNCH("ns_gram");
                if (p.split) { hipLaunchKernelGGL(ns_gram_finish_kernel, dim3((unsigned)p.sym), dim3(256), 0, st, tab, n, alpha); SAUNET_CHECK_LAUNCH("ns_gram_finish"); }
            }
            double q = 0;
            int Qb = NS_Q0;
            auto launch = [&](NsProds pr, int ny) { if (go) hipLaunchKernelGGL(ns_sym_kernel, dim3((unsigned)p.sym, ny), dim3(256), NsCore::LDS, st, tab, n, pr); };
            for (int j = 0; j < nb; ++j) {
                for (int i = 0; i <= NS_GRID; ++i) P[i] = b * S[i] + c * S[i] * S[i];
                sp = ns_scale(P);
                if (sp == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
                const int Pb = j ? NS_P : NS_Q0;
                launch(NsProds{{{NS_A, NS_A, NS_A, -1, Pb, (float)(c * sp / ((double)sa * sa)), (float)(b * sp / sa), 0.f}, {}}}, 1);
                NsProds pr = {};
                int ny = 0;
                if (j == 0) { for (int i = 0; i <= NS_GRID; ++i) Q[i] = P[i]; sq = sp; q = a; }
                else {
                    for (int i = 0; i <= NS_GRID; ++i) Q[i] = a * Q[i] + q * P[i] + P[i] * Q[i];
                    const float s2 = ns_scale(Q);
                    if (s2 == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
                    pr.p[ny++] = {NS_P, Qb, Qb, NS_P, Qb == NS_Q0 ? NS_Q1 : NS_Q0, (float)(s2 / ((double)sp * sq)), (float)(a * s2 / sq), (float)(q * s2 / sp)};
                    Qb = Qb == NS_Q0 ? NS_Q1 : NS_Q0; sq = s2; q *= a;
                }
                float sr = 0;
                if (j < nb - 1) {
                    for (int i = 0; i <= NS_GRID; ++i) R[i] = (a + P[i]) * S[i];
                    sr = ns_scale(R);
                    if (sr == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
                    pr.p[ny++] = {Pb, NS_A, NS_A, -1, NS_R, (float)(sr / ((double)sp * sa)), (float)(a * sr / sa), 0.f};
                }
                if (ny) launch(pr, ny);
                if (j < nb - 1) {
                    for (int i = 0; i <= NS_GRID; ++i) S[i] = (a + P[i]) * R[i];
                    const float s2 = ns_scale(S);
                    if (s2 == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
                    launch(NsProds{{{NS_R, Pb, NS_R, -1, NS_A, (float)(s2 / ((double)sr * sp)), (float)(a * s2 / sr), 0.f}, {}}}, 1);
                    sa = s2;
                }
                if (go) SAUNET_CHECK_LAUNCH("ns_sym");
            }
            for (int i = 0; i <= NS_GRID; ++i) x[i] = (q + Q[i]) * x[i];
            done += nb;
            const float s2 = ns_scale(x);
            if (done < d->steps) {
                if (s2 == 0.f) return set_error(SAUNET_UNSUPPORTED, "%s: the coefficients drive singular values out of range", who);
                if (go) hipLaunchKernelGGL((ns_apply_kernel<T, 0>), dim3((unsigned)p.app), dim3(256), NsCore::LDS, st, tab, n, Qb, xt, (float)(s2 / ((double)sq * sx)), (float)(q * s2 / sx), hyper, 0);
                xt ^= 1; sx = s2;
            } else if (go) {
                hipLaunchKernelGGL((ns_apply_kernel<T, MUON ? 2 : 1>), dim3((unsigned)p.app), dim3(256), NsCore::LDS, st, tab, n, Qb, xt, (float)(1.0 / ((double)sq * sx)), (float)(q / sx), hyper, d->adjust);
            }
            if (go) SAUNET_CHECK_LAUNCH("ns_apply");
        }
    }
    return SAUNET_OK;
}

}  // namespace saunet

using namespace saunet;

extern "C" {

int64_t saunet_newton_schulz_workspace(const saunet_ns_desc* d)
{
    NsPlan p;
    int rc = ns_check(d, "newton_schulz");
    if (!rc) rc = ns_plan(d, p, nullptr, nullptr);
    return rc ? rc : p.bytes;
}

int saunet_newton_schulz(const saunet_ns_desc* d, void* workspace, int64_t workspace_bytes, void* stream)
{
    int rc = ns_check(d, "newton_schulz");
    if (rc) return rc;
    for (int i = 0; i < d->count; ++i) if (!d->item[i].src || !d->item[i].dst) return set_error(SAUNET_BAD_SHAPE, "newton_schulz: matrix %d has no memory", i);
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == SAUNET_F32) return ns_run<float, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
    if (d->dtype == SAUNET_BF16) return ns_run<u16, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
    return ns_run<_Float16, false>(d, nullptr, workspace, workspace_bytes, st, "newton_schulz");
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
    return ns_run<float, true>(d, hyper, workspace, workspace_bytes, (hipStream_t)stream, "muon");
}

}  // extern "C"
