// lrb_muon.hip -- K10: the orthogonalised update of a list of weights (momentum, polynomial iteration, step), gfx950 only.
//
//   m <- beta m + (1 - beta) g;  u = (1 - beta) g + beta m  (nesterov), else m;  without a momentum buffer u = g
//   X = u / max(|u|_F, eps), taken with its short side as rows: n x m, n <= m
//   steps times:  A = X X^T,  B = b A + c A^2,  X <- a X + B X
//   p <- decay p + alpha X
//
// Bound: the matrix cores (2 n^2 m + 2 n^3 + 2 n^2 m multiply-adds a step, of the two symmetric products half).  The
// float32 matrix instructions run at 1/16 of the rate of the 16-bit ones, so every factor is held as TWO float16 numbers,
// hi = fp16(s v) and lo = fp16(s v - hi), and a product is three: hi hi + hi lo + lo hi, added up in float32.  What is left
// out (lo lo and the rounding of lo) is about 2^-23 of the value, i.e. the result is as exact as float32 products are:
// the polynomial stretches small singular values by up to a^steps (485 for the usual coefficients), so a 16-bit iteration
// would return noise where a gradient is of low rank.  s is a power of two for each matrix, step and factor, from a bound
// on the factor's largest singular value (the Frobenius norm bounds X by 1, the polynomial's extremes bound what follows):
// no entry can leave fp16's range whatever the coefficients or the size of u, and the entries use its upper end.
//
// All products are of the form C[i][j] = sum_k P[i][k] Q[j][k] with k contiguous in both: A = X X^T and A^2 = A A^T as they
// stand, B X from X's transpose, which the epilogue writes beside X.  One workgroup a T x T tile of C; of the symmetric
// products the tiles on and above the diagonal are computed and mirrored.  Tiles of all weights of a call share a launch.
#include <limits.h>
#include <math.h>
#include <string.h>

#include "lrb_device.h"

typedef _Float16 mu_h;
typedef mu_h mu_h8 __attribute__((ext_vector_type(8)));
typedef mu_h mu_h4 __attribute__((ext_vector_type(4)));
typedef float mu_f16 __attribute__((ext_vector_type(16)));

#define MU_ITEMS 16       // weights of one launch (their descriptors travel as kernel arguments)
#define MU_STEPS 32       // longest iteration
#define MU_COEF 5         // floats of the table for each matrix and step: kA, kB1, kB2, kX1, kX2
#define MU_TOP 57344.0    // the largest entry that a factor is scaled to: 7/8 of fp16's largest number
#define MU_BK 32          // k of one stage in LDS

struct mu_item {
    void *p;
    const void *g;
    void *m;
    long long ps[3], gs[3], ms[3]; // element strides of (matrix, short side, long side)
    unsigned long long off, step;  // bytes: the first matrix's planes in the workspace, from one matrix to the next
    int n, l, np, lp, count;       // short side, long side, both padded to 64; matrices
    int first;                     // number of the first matrix in the tables
    int p_type, g_type, m_type;
    float alpha, decay;
};

struct mu_args {
    char *ws;
    double *x0;     // [matrices] what u is multiplied by
    float *table;   // [matrices][steps][MU_COEF]
    double *part;   // [tiles of 64 x 64 of all matrices] sums of squares
    int n_items, steps;
    float beta, eps, a, b, c;
    int nesterov;
    int flip;       // which of the two copies of X is read
    int step;
    // of a product's launch: the tiles from `direct` on are cut along k, `splits` workgroups each, whose sums go to `parts`
    int direct, splits;
    float *parts;
    double sx;                      // the scale of X at the start, and the table, for a norm of at least eps
    float std[MU_STEPS * MU_COEF];
    int start[MU_ITEMS + 1]; // first tile of each item in this launch
    mu_item it[MU_ITEMS];
};
static_assert(sizeof(mu_args) <= 4096, "kernel arguments");

// The factors of a matrix: X and its transpose twice (read and written in turn), A, B, as rows of 32 hi, the 32 lo of the same
// entries, the next 32 hi ...: 32 k of a row are one whole line of 128 bytes, which halves the requests that the L2 gets for a
// stage against separate planes (2.1 -> 1.05 requests for 128 bytes).  And X and A in
// float32, for the terms a X and b A: hi + lo is a rounding more than float32 is, and these terms would pass it on.
__host__ __device__ inline unsigned long long mu_plane_x(const mu_item &it) { return 2ull * (unsigned long long)it.np * it.lp; }
__host__ __device__ inline unsigned long long mu_plane_a(const mu_item &it) { return 2ull * (unsigned long long)it.np * it.np; }
__host__ __device__ inline unsigned long long mu_bytes(const mu_item &it) { return 10 * mu_plane_x(it) + 6 * mu_plane_a(it); }

struct mu_mat {
    mu_h *x, *xt, *x2, *xt2, *a, *b;
    float *x32, *a32;
};
__device__ __forceinline__ mu_mat mu_planes(const mu_args &a, const mu_item &it, int mat)
{
    char *w = a.ws + it.off + (unsigned long long)mat * it.step;
    const unsigned long long px = 2 * mu_plane_x(it), pa = 2 * mu_plane_a(it);
    mu_mat r;
    r.x = (mu_h *)(w + (a.flip ? 2 * px : 0));
    r.xt = (mu_h *)(w + (a.flip ? 3 * px : px));
    r.x2 = (mu_h *)(w + (a.flip ? 0 : 2 * px));
    r.xt2 = (mu_h *)(w + (a.flip ? px : 3 * px));
    r.a = (mu_h *)(w + 4 * px);
    r.b = (mu_h *)(w + 4 * px + pa);
    r.x32 = (float *)(w + 4 * px + 2 * pa);
    r.a32 = (float *)(w + 5 * px + 2 * pa);
    return r;
}

// hi of entry (row, k) of a factor with rows of `len`; lo lies 32 further
__device__ __forceinline__ size_t mu_at(int row, int k, int len) { return (size_t)row * 2 * len + (k >> 5) * 64 + (k & 31); }

__device__ __forceinline__ float mu_load(const void *p, long long at, int type)
{
    return type == LRB_F32 ? ((const float *)p)[at] : type == LRB_BF16 ? (float)((const __bf16 *)p)[at] : (float)((const mu_h *)p)[at];
}
__device__ __forceinline__ void mu_store(void *p, long long at, int type, float v)
{
    if (type == LRB_F32) ((float *)p)[at] = v;
    else if (type == LRB_BF16) ((__bf16 *)p)[at] = (__bf16)v;
    else ((mu_h *)p)[at] = (mu_h)v;
}

// Which item a tile of the launch belongs to.
__device__ __forceinline__ int mu_find(const mu_args &a, int tile)
{
    int k = 0;
    while (k + 1 < a.n_items && tile >= a.start[k + 1]) ++k;
    return k;
}

// u at N places (row i(e), column j(e), where they lie inside), 0 elsewhere.  All loads are issued before the first result is
// used.  UPDATE also writes the momentum back (each entry by one thread).
template <bool UPDATE, int N, typename I, typename J>
__device__ __forceinline__ void mu_u(float beta, int nesterov, const mu_item &it, int mat, I i, J j, float (&u)[N])
{
    float m[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const bool in = i(e) < it.n && j(e) < it.l;
        u[e] = in ? mu_load(it.g, mat * it.gs[0] + i(e) * it.gs[1] + j(e) * it.gs[2], it.g_type) : 0.0f;
        m[e] = in && it.m ? mu_load(it.m, mat * it.ms[0] + i(e) * it.ms[1] + j(e) * it.ms[2], it.m_type) : 0.0f;
    }
    if (!it.m) return;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (UPDATE) {
            m[e] = beta * m[e] + (1.0f - beta) * u[e];
            if (i(e) < it.n && j(e) < it.l) mu_store(it.m, mat * it.ms[0] + i(e) * it.ms[1] + j(e) * it.ms[2], it.m_type, m[e]);
            // u is made of what is kept
            m[e] = it.m_type == LRB_F32 ? m[e] : it.m_type == LRB_BF16 ? (float)(__bf16)m[e] : (float)(mu_h)m[e];
        }
        u[e] = nesterov ? (1.0f - beta) * u[e] + beta * m[e] : m[e];
    }
}

// Momentum, and the sum of the squares of u over a 64 x 64 tile, in double (the squares of large float32 leave its range).
__global__ __launch_bounds__(256) void mu_momentum_kernel(mu_args a)
{
    __shared__ double red[4];
    const int k = mu_find(a, blockIdx.x);
    const mu_item &it = a.it[k];
    const int tj = it.lp / 64, per = (it.np / 64) * tj, local = blockIdx.x - a.start[k], mat = local / per, r = local % per;
    const int i0 = (r / tj) * 64, j0 = (r % tj) * 64;
    const bool along_j = it.gs[2] == 1 || it.gs[1] != 1;
    double s = 0.0;
    // entry e of a thread: 64 of a line by the lanes of a wave, four lines further for each e
    auto fast = [&](int) { return (int)(threadIdx.x & 63); };
    auto slow = [&](int e) { return e * 4 + (int)(threadIdx.x >> 6); };
    float u[16];
    if (along_j) mu_u<true>(a.beta, a.nesterov, it, mat, [&](int e) { return i0 + slow(e); }, [&](int e) { return j0 + fast(e); }, u);
    else mu_u<true>(a.beta, a.nesterov, it, mat, [&](int e) { return i0 + fast(e); }, [&](int e) { return j0 + slow(e); }, u);
#pragma unroll
    for (int e = 0; e < 16; ++e) s += (double)u[e] * u[e];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    lrb_barrier();
    if (threadIdx.x == 0) a.part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__host__ __device__ double mu_largest_odd(double a, double b, double c, double r) // max |a x + b x^3 + c x^5| over [0, r]
{
    double best = fabs(r * (a + r * r * (b + c * r * r)));
    const double d = 9.0 * b * b - 20.0 * a * c; // 5 c t^2 + 3 b t + a = 0, t = x^2
    for (int s = -1; s <= 1; s += 2) {
        const double t = c != 0.0 ? (d >= 0.0 ? (-3.0 * b + s * sqrt(d)) / (10.0 * c) : -1.0) : b != 0.0 ? -a / (3.0 * b) : -1.0;
        if (t > 0.0 && t < r * r) best = fmax(best, fabs(sqrt(t) * (a + t * (b + c * t))));
    }
    return best;
}

__host__ __device__ double mu_scale(double r) // the power of two that takes entries up to r to at most MU_TOP
{
    if (!(r > 0.0 && r < 1e300)) return 1.0;
    int e;
    frexp(MU_TOP / r, &e); // MU_TOP / r = f 2^e, 1/2 <= f < 1
    return ldexp(1.0, e - 1);
}

// The scale of X at the start, for singular values up to r, and the five factors of every step.
__host__ __device__ inline double mu_chain(double a, double b, double c, int steps, double r, float *t)
{
    const double slack = 1.0 + 1.0 / 512.0; // for the roundings on the way: the bounds hold for exact factors
    r *= slack;
    const double s0 = mu_scale(r);
    double sx = s0;
    for (int q = 0; q < steps; ++q, t += MU_COEF) {
        const double ra = r * r * slack, sa = mu_scale(ra);
        double rb = fabs(b * ra + c * ra * ra);
        if (c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < ra) rb = fmax(rb, b * b / fabs(4.0 * c));
        rb *= slack;
        const double sb = mu_scale(rb);
        r = mu_largest_odd(a, b, c, r) * slack;
        const double sn = q + 1 < steps ? mu_scale(r) : 1.0;
        t[0] = (float)(sa / (sx * sx));
        t[1] = (float)(b * (sb / sa));
        t[2] = (float)(c * (sb / sa) / sa);
        t[3] = (float)(a * (sn / sx));
        t[4] = (float)(sn / sb / sx);
        sx = sn;
    }
    return s0;
}

// From the sum of the squares of u: what u is multiplied by to become X, and the bound r on X's singular values.  At r = 1 the
// ready table holds.  An infinity or a NaN anywhere makes the whole matrix NaN.
struct mu_norm {
    double x0, r;
};
__device__ __forceinline__ mu_norm mu_start(double squares, double eps)
{
    const double norm = sqrt(squares), over = fmax(norm, eps);
    mu_norm n;
    n.r = !(norm < over) && norm > 0.0 ? 1.0 : fmax(norm / over, 1e-60);
    n.x0 = !(norm < 1e300) ? (double)NAN : over > 0.0 ? 1.0 / over : 0.0;
    return n;
}

// The norm of every matrix, and with it the scales of its factors in every step.
__global__ __launch_bounds__(256) void mu_table_kernel(mu_args a)
{
    __shared__ double red[4];
    int k = 0;
    while (k + 1 < a.n_items && (int)blockIdx.x >= a.it[k + 1].first) ++k;
    const mu_item &it = a.it[k];
    const int per = (it.np / 64) * (it.lp / 64), mat = blockIdx.x - it.first;
    const double *part = a.part + a.start[k] + (size_t)mat * per;
    double s = 0.0;
    for (int i = threadIdx.x; i < per; i += 256) s += part[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    lrb_barrier();
    const mu_norm n = mu_start(red[0] + red[1] + red[2] + red[3], a.eps);
    float *t = a.table + (size_t)blockIdx.x * a.steps * MU_COEF;
    if (n.r == 1.0 && (int)threadIdx.x < a.steps * MU_COEF) t[threadIdx.x] = a.std[threadIdx.x];
    if (threadIdx.x == 0) a.x0[blockIdx.x] = n.x0 * (n.r == 1.0 ? a.sx : mu_chain(a.a, a.b, a.c, a.steps, n.r, t));
}

__device__ __forceinline__ void mu_split(float v, mu_h &hi, mu_h &lo)
{
    hi = (mu_h)v;
    lo = (mu_h)(v - (float)hi);
}

// u, scaled and split, as X and as its transpose: a 64 x 64 tile through LDS, so that all sides are read and written in rows.
__global__ __launch_bounds__(256) void mu_split_kernel(mu_args a)
{
    __shared__ float tile[64][65];
    const int k = mu_find(a, blockIdx.x);
    const mu_item &it = a.it[k];
    const int tj = it.lp / 64, per = (it.np / 64) * tj, local = blockIdx.x - a.start[k], mat = local / per, r = local % per;
    const int i0 = (r / tj) * 64, j0 = (r % tj) * 64;
    const bool along_j = it.gs[2] == 1 || it.gs[1] != 1;
    const double scale = a.x0[it.first + mat];
    auto fast = [&](int) { return (int)(threadIdx.x & 63); };
    auto slow = [&](int e) { return e * 4 + (int)(threadIdx.x >> 6); };
    float u[16];
    if (along_j) mu_u<false>(a.beta, a.nesterov, it, mat, [&](int e) { return i0 + slow(e); }, [&](int e) { return j0 + fast(e); }, u);
    else mu_u<false>(a.beta, a.nesterov, it, mat, [&](int e) { return i0 + fast(e); }, [&](int e) { return j0 + slow(e); }, u);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const bool in = along_j ? i0 + slow(e) < it.n && j0 + fast(e) < it.l : i0 + fast(e) < it.n && j0 + slow(e) < it.l;
        tile[along_j ? slow(e) : fast(e)][along_j ? fast(e) : slow(e)] = in ? (float)(scale * u[e]) : 0.0f; // (the scale may be NaN)
    }
    lrb_barrier();
    const mu_mat w = mu_planes(a, it, mat);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int q = e * 256 + threadIdx.x, row = q >> 3, c = (q & 7) * 8;
        float v[8];
        mu_h8 hi, lo;
        const size_t at = mu_at(i0 + row, j0 + c, it.lp), at_t = mu_at(j0 + row, i0 + c, it.np);
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
            mu_h h, l;
            v[e8] = tile[row][c + e8];
            mu_split(v[e8], h, l);
            hi[e8] = h, lo[e8] = l;
        }
        __builtin_memcpy(w.x32 + (size_t)(i0 + row) * it.lp + j0 + c, v, 32);
        *(mu_h8 *)(w.x + at) = hi;
        *(mu_h8 *)(w.x + at + 32) = lo;
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
            mu_h h, l;
            mu_split(tile[c + e8][row], h, l);
            hi[e8] = h, lo[e8] = l;
        }
        *(mu_h8 *)(w.xt + at_t) = hi;
        *(mu_h8 *)(w.xt + at_t + 32) = lo;
    }
}

enum { MU_GRAM = 0, MU_POLY = 1, MU_APPLY = 2, MU_LAST = 3 };

__device__ __forceinline__ void mu_dma(const char *src, char *dst)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

__device__ __forceinline__ void mu_wave_sync() // LDS written by lanes of this wave is read by others of it
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0)
    __builtin_amdgcn_wave_barrier();
}

// p <- decay p + alpha v for up to four entries, `stride` apart
template <typename T> __device__ __forceinline__ void mu_update(const mu_item &it, long long at, long long stride, int count, float4 v)
{
    T *p = (T *)it.p + at;
    if (stride == 1 && count == 4) {
        T t[4];
        if (it.decay != 0.0f) {
            __builtin_memcpy(t, p, sizeof(t));
            v.x = it.decay * (float)t[0] + it.alpha * v.x, v.y = it.decay * (float)t[1] + it.alpha * v.y;
            v.z = it.decay * (float)t[2] + it.alpha * v.z, v.w = it.decay * (float)t[3] + it.alpha * v.w;
        } else {
            v.x *= it.alpha, v.y *= it.alpha, v.z *= it.alpha, v.w *= it.alpha;
        }
        t[0] = (T)v.x, t[1] = (T)v.y, t[2] = (T)v.z, t[3] = (T)v.w;
        __builtin_memcpy(p, t, sizeof(t));
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= count) break;
        const float x = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
        p[e * stride] = (T)((it.decay != 0.0f ? it.decay * (float)p[e * stride] : 0.0f) + it.alpha * x);
    }
}
__device__ __forceinline__ void mu_update4(const mu_item &it, long long at, long long stride, int count, float4 v)
{
    if (it.p_type == LRB_F32) mu_update<float>(it, at, stride, count, v);
    else if (it.p_type == LRB_BF16) mu_update<__bf16>(it, at, stride, count, v);
    else mu_update<mu_h>(it, at, stride, count, v);
}

// What becomes of 32 x 32 NI entries of a product, of which a wave holds the sums: acc[y][4 q + e] of a lane is row (lane & 31),
// column 32 y + 8 q + 4 (lane >> 5) + e.  They go through `lds` (32 rows of MU_PITCH) to be read, combined and written in
// whole row segments, and once more by columns for the mirrored or transposed side.
#define MU_PITCH(NI) (32 * (NI) + 4)
template <int MODE, int NI>
__device__ __forceinline__ void mu_strip(const mu_args &a, const mu_item &it, int mat, const mu_mat &w, const mu_f16 (&acc)[NI], int i0, int j0,
                                         bool mirror, float *lds, int lane)
{
    constexpr int PITCH = MU_PITCH(NI), LANES = 8 * NI, ROWS = 64 / LANES; // lanes of a row, rows of a turn
    const float *t = a.table + ((size_t)(it.first + mat) * a.steps + a.step) * MU_COEF;
    const float k1 = MODE == MU_GRAM ? 0.0f : MODE == MU_POLY ? t[1] : t[3], k2 = MODE == MU_GRAM ? t[0] : MODE == MU_POLY ? t[2] : t[4];
    const int ld = MODE >= MU_APPLY ? it.lp : it.np;
    float *full = MODE <= MU_POLY ? w.a32 : w.x32;
    mu_h *out = MODE == MU_GRAM ? w.a : MODE == MU_POLY ? w.b : w.x2, *out_t = MODE == MU_APPLY ? w.xt2 : out;
    const bool by_rows = it.ps[2] == 1 || it.ps[1] != 1; // which way p is written
    mu_wave_sync();
#pragma unroll
    for (int y = 0; y < NI; ++y)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *(float4 *)(lds + (lane & 31) * PITCH + 32 * y + 8 * q + 4 * (lane >> 5)) =
                make_float4(acc[y][4 * q], acc[y][4 * q + 1], acc[y][4 * q + 2], acc[y][4 * q + 3]);
    mu_wave_sync();
    const bool back = MODE == MU_LAST ? !by_rows : mirror;
#pragma unroll(MODE == MU_LAST ? 1 : 4)
    for (int r = lane / LANES; r < 32; r += ROWS) {
        const int c = (lane % LANES) * 4, i = i0 + r, j = j0 + c;
        if (i >= it.np || j >= ld) continue;
        float4 v = *(const float4 *)(lds + r * PITCH + c);
        float4 *const old = (float4 *)(full + (size_t)i * ld + j);
        const float4 o = MODE == MU_GRAM ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *old;
        v = make_float4(k1 * o.x + k2 * v.x, k1 * o.y + k2 * v.y, k1 * o.z + k2 * v.z, k1 * o.w + k2 * v.w);
        if (back) *(float4 *)(lds + r * PITCH + c) = v;
        if (MODE == MU_LAST) {
            if (by_rows && i < it.n && j < it.l) mu_update4(it, mat * it.ps[0] + i * it.ps[1] + j * it.ps[2], it.ps[2], min(4, it.l - j), v);
        } else {
            mu_h h0, h1, h2, h3, l0, l1, l2, l3;
            mu_split(v.x, h0, l0), mu_split(v.y, h1, l1), mu_split(v.z, h2, l2), mu_split(v.w, h3, l3);
            if (MODE != MU_POLY) *old = v; // B is a factor only
            *(mu_h4 *)(out + mu_at(i, j, ld)) = mu_h4{h0, h1, h2, h3};
            *(mu_h4 *)(out + mu_at(i, j, ld) + 32) = mu_h4{l0, l1, l2, l3};
        }
    }
    if (!back) return;
    mu_wave_sync();
#pragma unroll(MODE == MU_LAST ? 1 : 2 * NI)
    for (int s = 0; s < 2 * NI; ++s) {
        const int c = s * 16 + lane / 4, r = (lane % 4) * 8, i = i0 + r, j = j0 + c;
        if (i >= it.np || j >= ld) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lds[(r + e) * PITCH + c];
        if (MODE == MU_LAST) {
            if (j >= it.l) continue;
            const long long at = mat * it.ps[0] + i * it.ps[1] + j * it.ps[2];
            if (i < it.n) mu_update4(it, at, it.ps[1], min(4, it.n - i), make_float4(v[0], v[1], v[2], v[3]));
            if (i + 4 < it.n) mu_update4(it, at + 4 * it.ps[1], it.ps[1], min(4, it.n - i - 4), make_float4(v[4], v[5], v[6], v[7]));
        } else {
            mu_h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                mu_h h, l;
                mu_split(v[e], h, l);
                hi[e] = h, lo[e] = l;
            }
            *(mu_h8 *)(out_t + mu_at(j, i, it.np)) = hi;
            *(mu_h8 *)(out_t + mu_at(j, i, it.np) + 32) = lo;
        }
    }
}

// Where the tile with number `local` of a matrix lies, in tiles.  Four rows of tiles at a time, column by column: the tiles
// that an XCD has in flight together are as square a block as can be, so that its L2 serves most of their loads.
template <int MODE> __device__ __forceinline__ void mu_place(int local, int ti, int tj, int &i0, int &j0)
{
    i0 = 0, j0 = local;
    if (MODE >= MU_APPLY) {
        const int band = j0 / (4 * tj), h = min(4, ti - 4 * band);
        j0 -= band * 4 * tj;
        i0 = 4 * band + j0 % h;
        j0 /= h;
        return;
    }
    // the tiles on and above the diagonal: of each band first the triangle, then what lies right of it
    int h = min(4, ti);
    while (j0 >= h * (ti - i0) - h * (h - 1) / 2) {
        j0 -= h * (ti - i0) - h * (h - 1) / 2;
        i0 += 4;
        h = min(4, ti - i0);
    }
    const int band = i0, triangle = h * (h + 1) / 2;
    if (j0 < triangle) {
        int r = 0;
        while (j0 >= h - r) j0 -= h - r++;
        i0 = band + r;
        j0 += i0;
    } else {
        j0 -= triangle;
        i0 = band + j0 % h;
        j0 = band + h + j0 / h;
    }
}

// neighbouring workgroups go to different XCDs: each of the eight takes a run of neighbouring tiles
__device__ __forceinline__ int mu_by_xcd(int block, int total) { return (block & 7) * ((total + 7) / 8) + (block >> 3); }

// One tile of a product.  LDS holds two stages of 32 k: T rows of P and T of Q, 128 bytes each; the eight 16-byte chunks of a
// row (four of hi, four of lo) lie at chunk ^ ((row >> 1) & 7), which spreads the 16 rows that a quarter wave reads over all
// 64 banks.  The loads go from global memory to LDS directly, one stage ahead of the products.
template <int T, int WM, int WN, int MODE>
__global__ __launch_bounds__(64 * WM * WN) void mu_product_kernel(mu_args a)
{
    constexpr int WAVES = WM * WN, MI = T / WM / 32, NI = T / WN / 32;
    __shared__ __attribute__((aligned(1024))) char buf0[4 * T * 64];
    __shared__ __attribute__((aligned(1024))) char buf1[4 * T * 64];
    // first the workgroups of the whole tiles, then those of the tiles that are cut along k
    const int total = a.start[a.n_items], whole = (a.direct + 7) / 8 * 8, cut = total - a.direct;
    const int unit = (int)blockIdx.x < whole ? mu_by_xcd(blockIdx.x, a.direct) : mu_by_xcd(blockIdx.x - whole, cut * a.splits);
    const bool part = (int)blockIdx.x >= whole;
    if (unit >= (part ? cut * a.splits : a.direct)) return;
    const int tile = part ? a.direct + unit / a.splits : unit;
    const int k = mu_find(a, tile);
    const mu_item &it = a.it[k];
    const int ti = (it.np + T - 1) / T, tj = MODE >= MU_APPLY ? (it.lp + T - 1) / T : ti;
    const int per = MODE >= MU_APPLY ? ti * tj : ti * (ti + 1) / 2, local = tile - a.start[k], mat = local / per;
    int i0, j0;
    mu_place<MODE>(local % per, ti, tj, i0, j0);
    i0 *= T, j0 *= T;
    const mu_mat w = mu_planes(a, it, mat);
    const int K = MODE == MU_GRAM ? it.lp : it.np, jrows = MODE >= MU_APPLY ? it.lp : it.np;
    const mu_h *P = MODE == MU_GRAM ? w.x : MODE == MU_POLY ? w.a : w.b, *Q = MODE == MU_GRAM ? w.x : MODE == MU_POLY ? w.a : w.xt;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave / WN, wj = wave % WN;

    // A load of a wave fills eight rows of a stage.  All addresses are a factor's first row of the tile (uniform) and an offset of
    // the lane's row in it (32 bits: 256 rows of up to 2^22 entries); rows past the padding (tiles larger than 64) repeat the last
    // one, and what they give is not stored.
    constexpr int ROWS = WAVES * 8, FILLS = T / ROWS; // rows that the waves fill together; such fills of P, and of Q
    uint32_t off_p[FILLS], off_q[FILLS];
#pragma unroll
    for (int q = 0; q < FILLS; ++q) {
        const int row = q * ROWS + wave * 8 + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
        off_p[q] = (uint32_t)min(row, it.np - 1 - i0) * (uint32_t)K * 4 + chunk * 16;
        off_q[q] = (uint32_t)min(row, jrows - 1 - j0) * (uint32_t)K * 4 + chunk * 16;
    }
    // this workgroup's k, in units of 64
    const int units = K / 64, k_first = part ? (int)((long long)units * (unit % a.splits) / a.splits) * 64 : 0;
    const int k_end = part ? (int)((long long)units * (unit % a.splits + 1) / a.splits) * 64 : K;
    const char *const base_p = (const char *)(P + (size_t)i0 * 2 * K), *const base_q = (const char *)(Q + (size_t)j0 * 2 * K);

    mu_f16 acc[MI][NI];
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int y = 0; y < NI; ++y)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[x][y][v] = 0.0f;

    const int frow = lane & 31, fchunk = lane >> 5;
    auto stage = [&](char *buf, int k0) {
        const char *const p = base_p + 4 * (size_t)k0, *const q = base_q + 4 * (size_t)k0;
#pragma unroll
        for (int h = 0; h < FILLS; ++h) {
            mu_dma(p + off_p[h], buf + (h * ROWS + wave * 8) * 128);
            mu_dma(q + off_q[h], buf + (T + h * ROWS + wave * 8) * 128);
        }
        __builtin_amdgcn_sched_barrier(0); // else the compiler sinks the loads to the wait that ends the stage
    };
    struct frags {
        mu_h8 ph[MI], pl[MI], qh[NI], ql[NI];
    };
    // the chunk of a row does not depend on which 32 rows it is among: (row >> 1) & 7 == (frow >> 1) & 7
    const int at = frow * 128 + ((fchunk ^ ((frow >> 1) & 7)) << 4);
    auto read = [&](frags &f, const char *buf, int kk) {
        const char *const p = buf + wi * MI * 4096, *const q = buf + T * 128 + wj * NI * 4096;
        const int hi = at ^ (kk * 32), lo = hi ^ 64;
#pragma unroll
        for (int y = 0; y < NI; ++y) {
            f.qh[y] = *(const mu_h8 *)(q + y * 4096 + hi);
            f.ql[y] = *(const mu_h8 *)(q + y * 4096 + lo);
        }
#pragma unroll
        for (int x = 0; x < MI; ++x) {
            f.ph[x] = *(const mu_h8 *)(p + x * 4096 + hi);
            f.pl[x] = *(const mu_h8 *)(p + x * 4096 + lo);
        }
    };
    auto products = [&](const frags &f) {
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int y = 0; y < NI; ++y) {
                acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ql[y], f.ph[x], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.qh[y], f.pl[x], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.qh[y], f.ph[x], acc[x][y], 0, 0, 0);
            }
        // the reads of the next fragments, which are independent of these products, go between them
#pragma unroll
        for (int r = 0; r < 2 * (MI + NI); ++r) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); // an LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, 3 * MI * NI / (2 * (MI + NI)), 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 3 * MI * NI, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // K is a multiple of 64: two stages a turn, two times 16 k in each.  While the products of one fragment set run, the next set
    // is read; in the middle of a stage, when a wave has read all it needs of it, comes the barrier behind which the
    // stage's buffer is filled again -- by then the other buffer's loads, issued one stage ago, have arrived.  The last turns
    // load and read the last stage once more than needed: branches would part the reads from the products.
    frags f0, f1;
    auto turn = [&](char *buf, char *next, int k0) {
        read(f1, buf, 1);
        products(f0);
        __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0), lgkmcnt(0): the next stage is there, this one is read
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        stage(buf, min(k0 + 2 * MU_BK, k_end - MU_BK));
        read(f0, next, 0);
        products(f1);
    };
    stage(buf0, k_first);
    stage(buf1, k_first + MU_BK);
    __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
    lrb_barrier();
    read(f0, buf0, 0);
    for (int k0 = k_first; k0 < k_end; k0 += 2 * MU_BK) {
        turn(buf0, buf1, k0);
        turn(buf1, buf0, k0 + MU_BK);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lrb_barrier();

    if (part) { // the sums as they lie in the registers: mu_join_kernel adds them up
        float4 *const out = (float4 *)(a.parts + (size_t)unit * T * T) + (size_t)wave * MI * NI * 256 + lane;
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int y = 0; y < NI; ++y)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    out[((x * NI + y) * 4 + q) * 64] =
                        make_float4(acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2], acc[x][y][4 * q + 3]);
        return;
    }
    constexpr int HALF = WAVES / 2, LDS_WAVE = 32 * MU_PITCH(NI) * 4;
    static_assert(HALF * LDS_WAVE <= 4 * T * 64, "");
    float *const lds = (float *)((wave < HALF ? buf0 : buf1) + (wave % HALF) * LDS_WAVE);
    const bool mirror = MODE == MU_APPLY || i0 != j0;
#pragma unroll
    for (int x = 0; x < MI; ++x)
        mu_strip<MODE, NI>(a, it, mat, w, acc[x], i0 + (wi * MI + x) * 32, j0 + wj * NI * 32, mirror, lds, lane);
}

// The tiles that were cut along k: their parts' sums, added up in order, a wave for each 32 rows of one of the tile's waves.
template <int T, int WM, int WN, int MODE> __global__ __launch_bounds__(64) void mu_join_kernel(mu_args a)
{
    constexpr int WAVES = WM * WN, MI = T / WM / 32, NI = T / WN / 32;
    __shared__ float lds[32 * MU_PITCH(NI)];
    const int lane = threadIdx.x, r = blockIdx.x / (WAVES * MI), strip = blockIdx.x % (WAVES * MI), wave = strip / MI, x = strip % MI;
    const int tile = a.direct + r, k = mu_find(a, tile);
    const mu_item &it = a.it[k];
    const int ti = (it.np + T - 1) / T, tj = MODE >= MU_APPLY ? (it.lp + T - 1) / T : ti;
    const int per = MODE >= MU_APPLY ? ti * tj : ti * (ti + 1) / 2, local = tile - a.start[k], mat = local / per;
    int i0, j0;
    mu_place<MODE>(local % per, ti, tj, i0, j0);
    i0 *= T, j0 *= T;
    const int wi = wave / WN, wj = wave % WN;
    mu_f16 acc[NI];
#pragma unroll
    for (int y = 0; y < NI; ++y)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[y][v] = 0.0f;
    const float4 *in = (const float4 *)(a.parts + (size_t)r * a.splits * T * T) + (size_t)strip * NI * 256 + lane;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s, in += T * T / 4)
#pragma unroll
        for (int y = 0; y < NI; ++y)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = in[(y * 4 + q) * 64];
                acc[y][4 * q] += v.x, acc[y][4 * q + 1] += v.y, acc[y][4 * q + 2] += v.z, acc[y][4 * q + 3] += v.w;
            }
    const mu_mat w = mu_planes(a, it, mat);
    mu_strip<MODE, NI>(a, it, mat, w, acc, i0 + (wi * MI + x) * 32, j0 + wj * NI * 32, MODE == MU_APPLY || i0 != j0, lds, lane);
}

// A matrix that fits one workgroup's LDS (128 x 176, 64 x 448, 32 x 1,136 and less) goes through all its steps there, in one
// launch: X as rows of hi then lo, and A, then B, as rows of hi then lo; rows are 16 bytes longer than their entries, so that
// 16 of them start in different banks.  Each wave keeps its 32 x 32 tiles of X, and of A on and above the diagonal, in float32
// in registers from step to step.  X^T for B X is read from X by the transposing LDS read: of 16 lanes that address four
// rows of 16 entries it gives each lane a column's four.
// Bound: the matrix cores of one CU and the barriers (five a step).
#define MU_SMALL_WAVES 16
#define MU_SMALL_LDS (158 * 1024) // of 160 KB; the static arrays take the rest
#define MU_SMALL_TILES 3          // of X for a wave at most

__host__ __device__ inline int mu_small_n(int n) { return (n + 31) / 32 * 32; }
__host__ __device__ inline int mu_small_l(int l) { return (l + 15) / 16 * 16; }
static inline int mu_small_bytes(int n, int l) // 0: too large
{
    const long long np = mu_small_n(n), lp = mu_small_l(l), bytes = np * (4 * lp + 16) + np * (4 * np + 16);
    const long long tiles = np / 32 * ((lp + 31) / 32);
    return np <= 128 && bytes <= MU_SMALL_LDS && tiles <= MU_SMALL_TILES * MU_SMALL_WAVES ? (int)bytes : 0;
}

__device__ __forceinline__ mu_h4 mu_read_column(const char *p)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(mu_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
}

// hi and lo of four neighbouring entries
__device__ __forceinline__ void mu_put4(char *hi_at, char *lo_at, float v0, float v1, float v2, float v3, mu_h4 &hi, mu_h4 &lo)
{
    mu_h h0, h1, h2, h3, l0, l1, l2, l3;
    mu_split(v0, h0, l0), mu_split(v1, h1, l1), mu_split(v2, h2, l2), mu_split(v3, h3, l3);
    hi = mu_h4{h0, h1, h2, h3}, lo = mu_h4{l0, l1, l2, l3};
    *(mu_h4 *)hi_at = hi;
    *(mu_h4 *)lo_at = lo;
}

// tile (ti, tj) of a symmetric matrix of np rows, and its mirror image
__device__ __forceinline__ void mu_put_symmetric(char *A, int np, int ti, int tj, int lane, const mu_f16 &v)
{
    const int pa = 4 * np + 16, i = ti * 32 + (lane & 31), j = tj * 32 + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        mu_h4 hi, lo;
        char *const at = A + i * pa + 2 * (j + 8 * q);
        mu_put4(at, at + 2 * np, v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3], hi, lo);
        if (ti == tj) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            char *const to = A + (j + 8 * q + e) * pa + 2 * i;
            *(mu_h *)to = hi[e];
            *(mu_h *)(to + 2 * np) = lo[e];
        }
    }
}

// the product of 32 rows at p and 32 rows at q, of len entries each (lo behind hi)
__device__ __forceinline__ void mu_small_rows(const char *p, const char *q, int len, mu_f16 &acc)
{
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll 2
    for (int k0 = 0; k0 < len; k0 += 16, p += 32, q += 32) {
        const mu_h8 ph = *(const mu_h8 *)p, pl = *(const mu_h8 *)(p + 2 * len), qh = *(const mu_h8 *)q, ql = *(const mu_h8 *)(q + 2 * len);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql, ph, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, pl, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, ph, acc, 0, 0, 0);
    }
}

__global__ __launch_bounds__(64 * MU_SMALL_WAVES) void mu_small_kernel(mu_args by_value)
{
    // The arguments where they lie (the first one starts the kernel's argument segment): with this many uses of `by_value` the
    // compiler copies all 3.5 KB of it to every thread's scratch.
    const mu_args &a = *(const mu_args *)__builtin_amdgcn_kernarg_segment_ptr();
    extern __shared__ __attribute__((aligned(16))) char mu_lds[];
    __shared__ double red[MU_SMALL_WAVES];
    __shared__ float own[MU_STEPS * MU_COEF];
    int k = 0;
    while (k + 1 < a.n_items && (int)blockIdx.x >= a.it[k + 1].first) ++k;
    const mu_item &it = a.it[k];
    const int mat = blockIdx.x - it.first, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 31, half = lane >> 5; // of a fragment: its row, and which 8 of 16 k
    const int np = mu_small_n(it.n), lp = mu_small_l(it.l), nt = np / 32, tiles = nt * ((lp + 31) / 32);
    const int px = 4 * lp + 16, pa = 4 * np + 16;
    char *const X = mu_lds, *const A = mu_lds + np * px;

    // A wave's tiles of X, four neighbouring columns in every four registers.  They are read (and at the end written) in pieces of
    // four along the side on which g (p) is contiguous, and change hands through LDS, where X will be.
    double s = 0.0;
    const bool along_j = it.gs[2] == 1 || it.gs[1] != 1;
#pragma unroll 1
    for (int tile = wave; tile < tiles; tile += MU_SMALL_WAVES) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int line = 8 * q + lane / 8, at = lane % 8 * 4;
            const int i = tile % nt * 32 + (along_j ? line : at), j = tile / nt * 32 + (along_j ? at : line);
            float u[4];
            if (along_j) mu_u<true>(a.beta, a.nesterov, it, mat, [&](int) { return i; }, [&](int e) { return j + e; }, u);
            else mu_u<true>(a.beta, a.nesterov, it, mat, [&](int e) { return i + e; }, [&](int) { return j; }, u);
#pragma unroll
            for (int e = 0; e < 4; ++e) s += (double)u[e] * u[e];
            if (j >= lp) continue; // (a piece lies within lp or outside)
            if (along_j) {
                *(float4 *)(X + i * px + 4 * j) = make_float4(u[0], u[1], u[2], u[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) *(float *)(X + (i + e) * px + 4 * j) = u[e];
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    lrb_barrier();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < MU_SMALL_WAVES; ++w) s += red[w];
    const mu_norm n = mu_start(s, a.eps);
    double x0 = n.x0;
    if (n.r == 1.0) { // (all threads have the same s)
        if ((int)threadIdx.x < a.steps * MU_COEF) own[threadIdx.x] = a.std[threadIdx.x];
        x0 *= a.sx;
    } else { // a norm below eps
        lrb_barrier(); // red has been read
        if (threadIdx.x == 0) red[0] = mu_chain(a.a, a.b, a.c, a.steps, n.r, own);
        lrb_barrier();
        x0 *= red[0];
    }
    const float *coef = own;
    float x[MU_SMALL_TILES][16];
#pragma unroll
    for (int t = 0; t < MU_SMALL_TILES; ++t) {
        const int tile = wave + t * MU_SMALL_WAVES;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = tile % nt * 32 + row, j = tile / nt * 32 + 4 * half + 8 * q;
            const float4 v = tile < tiles && j < lp ? *(const float4 *)(X + i * px + 4 * j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            x[t][4 * q] = (float)(x0 * v.x), x[t][4 * q + 1] = (float)(x0 * v.y);
            x[t][4 * q + 2] = (float)(x0 * v.z), x[t][4 * q + 3] = (float)(x0 * v.w);
        }
    }

    lrb_barrier(); // all have read: what follows writes hi and lo there
    // the wave's tile of the symmetric products, on or above the diagonal
    int ti = 0, tj = wave;
    while (ti < nt && tj >= nt - ti) tj -= nt - ti++;
    tj += ti;
    const bool sym = ti < nt;
    for (int step = 0; step < a.steps; ++step, coef += MU_COEF) {
        // the addresses below are made anew in every step: kept over the steps, all of them together spill
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int row = lane & 31, half = lane >> 5;
#pragma unroll
        for (int t = 0; t < MU_SMALL_TILES; ++t) {
            const int tile = wave + t * MU_SMALL_WAVES, i = tile % nt * 32 + row, j = tile / nt * 32 + 4 * half;
            if (tile >= tiles) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (j + 8 * q >= lp) continue;
                mu_h4 hi, lo;
                char *const at = X + i * px + 2 * (j + 8 * q);
                mu_put4(at, at + 2 * lp, x[t][4 * q], x[t][4 * q + 1], x[t][4 * q + 2], x[t][4 * q + 3], hi, lo);
            }
        }
        lrb_barrier();
        mu_f16 full, acc;
        if (sym) {
            mu_small_rows(X + (ti * 32 + row) * px + 16 * half, X + (tj * 32 + row) * px + 16 * half, lp, full);
#pragma unroll
            for (int e = 0; e < 16; ++e) full[e] *= coef[0];
            mu_put_symmetric(A, np, ti, tj, lane, full);
        }
        lrb_barrier();
        if (sym) {
            mu_small_rows(A + (ti * 32 + row) * pa + 16 * half, A + (tj * 32 + row) * pa + 16 * half, np, acc);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = coef[1] * full[e] + coef[2] * acc[e];
        }
        lrb_barrier();
        if (sym) mu_put_symmetric(A, np, ti, tj, lane, acc);
        lrb_barrier();
#pragma unroll
        for (int t = 0; t < MU_SMALL_TILES; ++t) {
            const int tile = wave + t * MU_SMALL_WAVES;
            if (tile >= tiles) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
            const char *p = A + (tile % nt * 32 + row) * pa + 16 * half;
            // rows k of X, 16 columns of the tile for each 16 lanes; columns past the end give what is not kept
            const char *q = X + (8 * half + (lane & 15) / 4) * px + 2 * (tile / nt * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
#pragma unroll 2
            for (int k0 = 0; k0 < np; k0 += 16, p += 32, q += 16 * px) {
                const mu_h8 ph = *(const mu_h8 *)p, pl = *(const mu_h8 *)(p + 2 * np);
                const mu_h4 h0 = mu_read_column(q), h1 = mu_read_column(q + 4 * px), l0 = mu_read_column(q + 2 * lp),
                            l1 = mu_read_column(q + 4 * px + 2 * lp);
                const mu_h8 qh = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7), ql = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql, ph, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, pl, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, ph, acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) x[t][e] = coef[3] * x[t][e] + coef[4] * acc[e];
        }
        lrb_barrier();
    }
#pragma unroll
    for (int t = 0; t < MU_SMALL_TILES; ++t) {
        const int tile = wave + t * MU_SMALL_WAVES;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = tile % nt * 32 + row, j = tile / nt * 32 + 4 * half + 8 * q;
            if (tile < tiles && j < lp) *(float4 *)(X + i * px + 4 * j) = make_float4(x[t][4 * q], x[t][4 * q + 1], x[t][4 * q + 2], x[t][4 * q + 3]);
        }
    }
    mu_wave_sync();
    const bool by_rows = it.ps[2] == 1 || it.ps[1] != 1;
#pragma unroll 1
    for (int tile = wave; tile < tiles; tile += MU_SMALL_WAVES) {
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
            const int line = 8 * q + lane / 8, at = lane % 8 * 4;
            const int i = tile % nt * 32 + (by_rows ? line : at), j = tile / nt * 32 + (by_rows ? at : line);
            if (i >= it.n || j >= it.l) continue;
            const char *v = X + i * px + 4 * j;
            const int step = by_rows ? 4 : px;
            const float4 f = make_float4(*(const float *)v, *(const float *)(v + step), *(const float *)(v + 2 * step), *(const float *)(v + 3 * step));
            mu_update4(it, mat * it.ps[0] + i * it.ps[1] + j * it.ps[2], by_rows ? it.ps[2] : it.ps[1], min(4, by_rows ? it.l - j : it.n - i), f);
        }
    }
}

// How a product's launch is laid out.
struct mu_plan {
    int T;             // side of a tile
    long long tiles;
    int direct, splits; // the first `direct` tiles are whole, the others are cut into `splits` along k
    uint64_t part_bytes() const { return splits > 1 ? (uint64_t)(tiles - direct) * splits * T * T * 4 : 0; }
};

static long long mu_tiles(const mu_args &a, bool symmetric, int T, int *start)
{
    long long sum = 0;
    for (int k = 0; k < a.n_items; ++k) {
        if (start) start[k] = (int)sum;
        const long long ti = (a.it[k].np + T - 1) / T, tj = (a.it[k].lp + T - 1) / T;
        sum += a.it[k].count * (symmetric ? ti * (ti + 1) / 2 : ti * tj);
    }
    if (start) start[a.n_items] = (int)sum;
    return sum;
}

// The tile: the largest that still gives most of the 256 CUs one (a larger tile loads less for each product).  Both symmetric
// products take the same (A in float32 is there on and above the diagonal's tiles only).
// The cut: a CU holds one, two or four workgroups by their LDS, so 256, 512 or 1024 tiles run side by side and take the same
// time; the tiles of the last, unfilled round are cut along k so that all CUs share them.
static mu_plan mu_lay_out(const mu_args &a, int mode)
{
    const bool symmetric = mode <= MU_POLY;
    mu_plan p;
    p.T = mu_tiles(a, symmetric, 256, nullptr) >= 200 ? 256 : mu_tiles(a, symmetric, 128, nullptr) >= 200 ? 128 : 64;
    p.tiles = mu_tiles(a, symmetric, p.T, nullptr);
    const int slots = p.T == 256 ? 256 : p.T == 128 ? 512 : 1024;
    const long long rest = p.tiles % slots;
    p.direct = (int)p.tiles, p.splits = 1;
    if (rest == 0) return p;
    long long units = 1ll << 40; // of 64 k, in the shortest of the rest's products
    long long before = 0;
    for (int k = 0; k < a.n_items; ++k) {
        const long long ti = (a.it[k].np + p.T - 1) / p.T, tj = (a.it[k].lp + p.T - 1) / p.T;
        before += a.it[k].count * (symmetric ? ti * (ti + 1) / 2 : ti * tj);
        const long long u = (mode == MU_GRAM ? a.it[k].lp : a.it[k].np) / 64;
        if (before > p.tiles - rest && u < units) units = u;
    }
    long long s = slots / rest;
    if (s > units / 4) s = units / 4; // 256 k a part at least
    if (s < 2 || units - units / s < 8) return p; // what is saved would not pay for the joining launch
    p.direct = (int)(p.tiles - rest), p.splits = (int)s;
    return p;
}

template <int T, int WM, int WN, int MODE> static void mu_launch_tiles(const mu_args &a, const mu_plan &p, hipStream_t st)
{
    const long long cut = p.tiles - p.direct, units = cut * p.splits;
    hipLaunchKernelGGL((mu_product_kernel<T, WM, WN, MODE>), dim3((unsigned)((p.direct + 7) / 8 * 8 + (units + 7) / 8 * 8)), dim3(64 * WM * WN), 0, st, a);
    if (cut) hipLaunchKernelGGL((mu_join_kernel<T, WM, WN, MODE>), dim3((unsigned)(cut * (T / 32) * WN)), dim3(64), 0, st, a);
}

template <int MODE> static void mu_launch_product(mu_args &a, hipStream_t st)
{
    const mu_plan p = mu_lay_out(a, MODE);
    mu_tiles(a, MODE <= MU_POLY, p.T, a.start);
    a.direct = p.direct, a.splits = p.splits;
    if (p.T == 256) mu_launch_tiles<256, 2, 4, MODE>(a, p, st);
    else if (p.T == 128) mu_launch_tiles<128, 2, 2, MODE>(a, p, st);
    else mu_launch_tiles<64, 2, 2, MODE>(a, p, st);
}

// A run of items (or of some matrices of one) that fits the descriptors and MU_WS_MOST bytes, and what it takes.
#define MU_WS_MOST (4ull << 30)
#define MU_MATS_MOST 4096
struct mu_group {
    mu_args a;
    int lds; // of a group whose matrices fit a workgroup's LDS: the most that one takes; else 0
    int mats;
    long long tiles;
    uint64_t planes;
    uint64_t bytes() const
    {
        if (lds) return 0;
        uint64_t parts = 0;
        for (int mode = MU_GRAM; mode <= MU_LAST; ++mode) {
            const uint64_t b = mu_lay_out(a, mode).part_bytes();
            parts = b > parts ? b : parts;
        }
        return planes + parts + ((uint64_t)mats * 8 + 255) / 256 * 256 + ((uint64_t)tiles * 8 + 255) / 256 * 256 +
               ((uint64_t)mats * MU_STEPS * MU_COEF * 4 + 255) / 256 * 256;
    }
};

// Calls `go(group)` for each group of the list in turn, those of small matrices first; stops at its first non-zero answer.
template <typename F> static int mu_each_group(const lrb_muon_item *items, int n_items, F go)
{
    for (int small = 1; small >= 0; --small) {
        mu_group gr = {};
        for (int k = 0; k < n_items; ++k) {
            const lrb_muon_item &s = items[k];
            if (s.count <= 0 || s.rows <= 0 || s.cols <= 0) continue;
            const bool turned = s.rows > s.cols;
            mu_item it = {};
            it.n = (int)(turned ? s.cols : s.rows), it.l = (int)(turned ? s.rows : s.cols);
            const int lds = mu_small_bytes(it.n, it.l);
            if ((lds != 0) != (small != 0)) continue;
            it.np = (it.n + 63) / 64 * 64, it.lp = (it.l + 63) / 64 * 64;
            it.step = mu_bytes(it);
            for (int d = 0; d < 3; ++d) {
                const int from = d && turned ? 3 - d : d;
                it.ps[d] = s.p_stride[from], it.gs[d] = s.g_stride[from], it.ms[d] = s.m_stride[from];
            }
            it.p_type = s.p_type, it.g_type = s.g_type, it.m_type = s.m_type;
            it.alpha = s.alpha, it.decay = s.decay;
            const long long per = (long long)(it.np / 64) * (it.lp / 64);
            const int size_p = s.p_type == LRB_F32 ? 4 : 2, size_g = s.g_type == LRB_F32 ? 4 : 2, size_m = s.m_type == LRB_F32 ? 4 : 2;
            for (int64_t done = 0; done < s.count;) {
                int64_t room = (1 << 20) - gr.mats;
                if (!small) {
                    room = gr.planes < MU_WS_MOST ? (int64_t)((MU_WS_MOST - gr.planes) / it.step) : 0;
                    if (room == 0 && gr.a.n_items == 0) room = 1;
                    if (room > MU_MATS_MOST - gr.mats) room = MU_MATS_MOST - gr.mats;
                    if (per * room > (1 << 28) - gr.tiles && room > 1) room = ((1 << 28) - gr.tiles) / per;
                }
                if (room == 0 || gr.a.n_items == MU_ITEMS) {
                    if (int rc = go(gr)) return rc;
                    gr = {};
                    continue;
                }
                it.count = (int)(s.count - done < room ? s.count - done : room);
                it.p = (char *)s.p + done * s.p_stride[0] * size_p;
                it.g = (const char *)s.g + done * s.g_stride[0] * size_g;
                it.m = s.m ? (char *)s.m + done * s.m_stride[0] * size_m : nullptr;
                it.off = gr.planes, it.first = gr.mats;
                gr.a.start[gr.a.n_items] = (int)gr.tiles;
                gr.a.it[gr.a.n_items++] = it;
                gr.mats += it.count;
                if (small) {
                    gr.lds = gr.lds > lds ? gr.lds : lds;
                } else {
                    gr.planes += it.step * it.count, gr.tiles += per * it.count;
                }
                gr.a.start[gr.a.n_items] = (int)gr.tiles;
                done += it.count;
            }
        }
        if (gr.a.n_items)
            if (int rc = go(gr)) return rc;
    }
    return LRB_OK;
}

static bool mu_items_fit(const lrb_muon_item *items, int n)
{
    for (int k = 0; k < n; ++k) {
        const lrb_muon_item &s = items[k];
        if (s.count < 0 || s.rows < 0 || s.cols < 0) return false;
        if (s.count == 0 || s.rows == 0 || s.cols == 0) continue;
        // a side below 2^22 and planes below 2^31 entries: the kernels' 32-bit indices hold
        if (s.rows > (1 << 22) || s.cols > (1 << 22) || (s.rows + 63) * (s.cols + 63) > INT_MAX) return false;
        if (!s.p || !s.g || s.p_type < LRB_F32 || s.p_type > LRB_F16 || s.g_type < LRB_F32 || s.g_type > LRB_F16) return false;
        if (s.m && (s.m_type < LRB_F32 || s.m_type > LRB_F16)) return false;
    }
    return true;
}

extern "C" double lrb_muon_bound(int steps, float a, float b, float c)
{
    double r = 1.0, most = 1.0;
    for (int k = 0; k < steps && k < MU_STEPS && r <= 1e9; ++k) {
        r = mu_largest_odd(a, b, c, r);
        most = most >= r ? most : r; // a NaN stays
    }
    return most;
}

extern "C" uint64_t lrb_muon_ws_bytes(const lrb_muon_item *items, int n_items)
{
    if (n_items <= 0 || !items || !mu_items_fit(items, n_items)) return 0;
    uint64_t most = 0;
    mu_each_group(items, n_items, [&](mu_group &gr) {
        if (gr.bytes() > most) most = gr.bytes();
        return LRB_OK;
    });
    return most;
}

extern "C" int lrb_muon_dev(int device, void *stream, const lrb_muon_item *items, int n_items, float momentum, int nesterov, int steps,
                            float a, float b, float c, float eps, void *d_ws, uint64_t ws_bytes)
{
    ARG_TRY(n_items >= 0 && (n_items == 0 || items != nullptr));
    ARG_TRY(steps >= 1 && steps <= MU_STEPS && eps >= 0.0f);
    ARG_TRY(lrb_muon_bound(steps, a, b, c) <= LRB_MUON_DIVERGED);
    ARG_TRY(mu_items_fit(items, n_items));
    const uint64_t need = lrb_muon_ws_bytes(items, n_items);
    ARG_TRY(need == 0 || (d_ws != nullptr && ws_bytes >= need && ((uintptr_t)d_ws & 255) == 0));
    bool any = false;
    for (int k = 0; k < n_items; ++k) any |= items[k].count > 0 && items[k].rows > 0 && items[k].cols > 0;
    if (!any) return LRB_OK;
    lrb_on_device on(device);
    HIP_TRY(on.err);
    hipStream_t st = (hipStream_t)stream;
    float std[MU_STEPS * MU_COEF] = {};
    const double sx = mu_chain(a, b, c, steps, 1.0, std);
    return mu_each_group(items, n_items, [&](mu_group &gr) -> int {
        mu_args &g = gr.a;
        g.steps = steps, g.beta = momentum, g.nesterov = nesterov, g.eps = eps, g.a = a, g.b = b, g.c = c;
        g.sx = sx;
        memcpy(g.std, std, sizeof(std));
        if (gr.lds) {
            static lrb_per_device_once raised;
            if (raised.need(device)) {
                HIP_TRY(hipFuncSetAttribute((const void *)mu_small_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, MU_SMALL_LDS));
            }
            hipLaunchKernelGGL(mu_small_kernel, dim3(gr.mats), dim3(64 * MU_SMALL_WAVES), gr.lds, st, g);
            HIP_TRY(hipGetLastError());
            return LRB_OK;
        }
        g.ws = (char *)d_ws;
        char *at = g.ws + gr.planes;
        g.x0 = (double *)at, at += ((uint64_t)gr.mats * 8 + 255) / 256 * 256;
        g.part = (double *)at, at += ((uint64_t)gr.tiles * 8 + 255) / 256 * 256;
        g.table = (float *)at, at += ((uint64_t)gr.mats * MU_STEPS * MU_COEF * 4 + 255) / 256 * 256;
        g.parts = (float *)at;
        hipLaunchKernelGGL(mu_momentum_kernel, dim3((unsigned)gr.tiles), dim3(256), 0, st, g);
        hipLaunchKernelGGL(mu_table_kernel, dim3(gr.mats), dim3(256), 0, st, g);
        hipLaunchKernelGGL(mu_split_kernel, dim3((unsigned)gr.tiles), dim3(256), 0, st, g);
        for (int s = 0; s < steps; ++s) {
            g.step = s;
            mu_launch_product<MU_GRAM>(g, st);
            mu_launch_product<MU_POLY>(g, st);
            if (s + 1 < steps) mu_launch_product<MU_APPLY>(g, st);
            else mu_launch_product<MU_LAST>(g, st);
            g.flip ^= 1;
        }
        HIP_TRY(hipGetLastError());
        return LRB_OK;
    });
}
