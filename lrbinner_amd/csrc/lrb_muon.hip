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
// Every step forms A from the X before it, for every type of p: a 16-bit result is the float32 result, rounded.  (Where X is longer
// than wide fewer products would do if A were carried over several steps by the polynomial it goes through; the rounding
// errors of the small singular values' part of A would then grow by a^2 a step instead of a.)  A matrix that fits one workgroup's LDS
// goes through all steps in one launch (mu_small_kernel).
// Measured, where a library product of 8192 x 8192 float16 reaches 1.09 PFLOP/s: a 4096 x 4096 float32 weight 3.9 ms = 1.05
// PFLOP/s of its three products (B X alone 1.14); a layer's four weights (2048 x 2048 twice, 5461 x 2048, 2048 x 5461,
// bfloat16) 3.99 ms, of them 0.17 for the momentum and the splitting, at 4.5 and 5.5 TB/s; 8 x 1024 x 2048 1.31 ms;
// 1025 x 511 158 us (23 launches that wait for each other); 128 x 168 51 us.
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "lrb_device.h"

typedef _Float16 mu_h;
typedef mu_h mu_h8 __attribute__((ext_vector_type(8)));
typedef mu_h mu_h4 __attribute__((ext_vector_type(4)));
typedef float mu_f16 __attribute__((ext_vector_type(16)));

#define MU_ITEMS 14       // weights of one launch (their descriptors travel as kernel arguments)
#define MU_STEPS 32       // longest iteration
#define MU_COEF 2         // factors of an operation: of the old entry, and of the sum of products
#define MU_OPS 3          // operations of a step
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
    double *x0;     // [matrices][2] what u is multiplied by; 1 if the launch's own factors hold, 0 for those of the table
    float *table;   // [matrices][steps][MU_OPS][MU_COEF]
    double *part;   // [tiles of 64 x 64 of all matrices] sums of squares
    int n_items, steps;
    float beta, rest; // the momentum, and 1 - momentum rounded by itself: 1 - beta of 0.999 would be off by 1e-5 of it
    float eps, a, b, c;
    int nesterov;
    int flip;       // which of the two copies of X is read
    int op;         // the operation of this launch, counted through the steps, and its factors for a norm of at least eps
    float k[MU_COEF];
    // of a product's launch: the tiles from `direct` on are cut along k, `splits` workgroups each, whose sums go to `parts`
    int direct, splits;
    float *parts;
    double sx;                       // the scale of X at the start for a norm of at least eps
    float std[MU_STEPS * MU_OPS * MU_COEF]; // and all factors
    int start[MU_ITEMS + 1]; // first tile of each item in this launch
    mu_item it[MU_ITEMS];
};
static_assert(sizeof(mu_args) <= 4096, "kernel arguments");

// A matrix in the workspace: X and its transpose twice (read and written in turn), A and B, as rows of 32 hi, the 32 lo of the
// same entries, the next 32 hi ...: 32 k of a row are one whole line of 128 bytes, which halves the requests that the L2 gets for
// a stage against separate planes of hi and lo (4096 x 4096, B X: 43 M -> 21 M).  And X and A in float32, for the terms that are
// not products (a X, b A): hi + lo is a rounding more than float32 is, and these terms would pass it on.  A's float32 is there on
// and above the diagonal's tiles.
__host__ __device__ inline unsigned long long mu_plane_x(const mu_item &it) { return 4ull * (unsigned long long)it.np * it.lp; }
__host__ __device__ inline unsigned long long mu_plane_a(const mu_item &it) { return 4ull * (unsigned long long)it.np * it.np; }
__host__ __device__ inline unsigned long long mu_bytes(const mu_item &it) { return 5 * mu_plane_x(it) + 3 * mu_plane_a(it); }

struct mu_mat {
    mu_h *x, *xt, *x2, *xt2, *a, *b;
    float *x32, *a32;
};
__device__ __forceinline__ mu_mat mu_planes(const mu_args &a, const mu_item &it, int mat)
{
    char *w = a.ws + it.off + (unsigned long long)mat * it.step;
    const unsigned long long px = mu_plane_x(it), pa = mu_plane_a(it);
    mu_mat r;
    r.x = (mu_h *)(w + (a.flip ? 2 * px : 0));
    r.xt = (mu_h *)(w + (a.flip ? 3 * px : px));
    r.x2 = (mu_h *)(w + (a.flip ? 0 : 2 * px));
    r.xt2 = (mu_h *)(w + (a.flip ? px : 3 * px));
    r.x32 = (float *)(w + 4 * px);
    r.a = (mu_h *)(w + 5 * px);
    r.b = (mu_h *)(w + 5 * px + pa);
    r.a32 = (float *)(w + 5 * px + 2 * pa);
    return r;
}

// hi of entry (row, k) of a factor with rows of `len`; lo lies 32 further
__device__ __forceinline__ size_t mu_at(int row, int k, int len) { return (size_t)row * 2 * len + (k >> 5) * 64 + (k & 31); }

// Which item a tile of the launch belongs to.
__device__ __forceinline__ int mu_find(const mu_args &a, int tile)
{
    int k = 0;
    while (k + 1 < a.n_items && tile >= a.start[k + 1]) ++k;
    return k;
}

// R pieces of four entries, `step` apart, of which `count(r)` lie inside (the others are 0): entry e of piece r is at
// at + r * piece + e * step.  The type is asked for once, so all pieces are on their way together.
template <typename T, int R, typename C>
__device__ __forceinline__ void mu_read(const T *p, long long at, long long piece, long long step, C count, float (&v)[4 * R])
{
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T *const q = p + at + r * piece;
        const int n = count(r);
        if (step == 1 && n == 4) {
            T t[4];
            __builtin_memcpy(t, q, sizeof(t));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * r + e] = (float)t[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * r + e] = e < n ? (float)q[e * step] : 0.0f;
        }
    }
}
template <int R, typename C>
__device__ __forceinline__ void mu_read(const void *p, int type, long long at, long long piece, long long step, C count, float (&v)[4 * R])
{
    if (type == LRB_F32) mu_read<float, R>((const float *)p, at, piece, step, count, v);
    else if (type == LRB_BF16) mu_read<__bf16, R>((const __bf16 *)p, at, piece, step, count, v);
    else mu_read<mu_h, R>((const mu_h *)p, at, piece, step, count, v);
}
template <typename T, int R, typename C>
__device__ __forceinline__ void mu_write(T *p, long long at, long long piece, long long step, C count, float (&v)[4 * R])
{
#pragma unroll
    for (int r = 0; r < R; ++r) {
        T *const q = p + at + r * piece;
        const int n = count(r);
        T t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            t[e] = (T)v[4 * r + e];
            v[4 * r + e] = (float)t[e]; // what is kept
        }
        if (step == 1 && n == 4) {
            __builtin_memcpy(q, t, sizeof(t));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) q[e * step] = t[e];
        }
    }
}

// u in R pieces of four along the side on which g is contiguous: piece r lies in line `line(r)` of the other side, from `at` on.
// UPDATE also writes the momentum back (each entry by one thread); u is made of what is kept.
template <bool UPDATE, int R, typename L>
__device__ __forceinline__ void mu_u(float beta, float rest, int nesterov, const mu_item &it, int mat, bool along_j, L line, int at, float (&u)[4 * R])
{
    const int lines = along_j ? it.n : it.l, len = along_j ? it.l : it.n;
    const long long g_fast = along_j ? it.gs[2] : it.gs[1], g_slow = along_j ? it.gs[1] : it.gs[2];
    const long long m_fast = along_j ? it.ms[2] : it.ms[1], m_slow = along_j ? it.ms[1] : it.ms[2];
    auto count = [=](int r) { return line(r) < lines ? max(0, min(4, len - at)) : 0; };
    const long long gap = R > 1 ? line(1) - line(0) : 0; // lines are evenly spaced
    mu_read<R>(it.g, it.g_type, mat * it.gs[0] + line(0) * g_slow + at * g_fast, gap * g_slow, g_fast, count, u);
    if (!it.m) return;
    float m[4 * R];
    const long long m_at = mat * it.ms[0] + line(0) * m_slow + at * m_fast;
    mu_read<R>(it.m, it.m_type, m_at, gap * m_slow, m_fast, count, m);
    if (UPDATE) {
#pragma unroll
        for (int e = 0; e < 4 * R; ++e) m[e] = beta * m[e] + rest * u[e];
        if (it.m_type == LRB_F32) mu_write<float, R>((float *)it.m, m_at, gap * m_slow, m_fast, count, m);
        else if (it.m_type == LRB_BF16) mu_write<__bf16, R>((__bf16 *)it.m, m_at, gap * m_slow, m_fast, count, m);
        else mu_write<mu_h, R>((mu_h *)it.m, m_at, gap * m_slow, m_fast, count, m);
    }
#pragma unroll
    for (int e = 0; e < 4 * R; ++e) u[e] = nesterov ? rest * u[e] + beta * m[e] : m[e];
}

// v times a double, rounded once or nearly so (to 2^-24 (1 + 2^-23)) without double arithmetic for each entry: the factor is
// (hi + lo) 2^e with 1/2 <= hi < 1.
struct mu_factor {
    float hi, lo;
    int e;
    __device__ __forceinline__ explicit mu_factor(double f)
    {
        const double m = frexp(f, &e); // a NaN or a zero stays
        hi = (float)m, lo = (float)(m - hi);
    }
    __device__ __forceinline__ float operator*(float v) const
    {
        const float w = ldexpf(v, e);
        return fmaf(w, hi, w * lo);
    }
};

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
    // sixteen threads a line of 64, four lines of a thread 16 apart
    float u[16];
    const int line = (along_j ? i0 : j0) + (threadIdx.x >> 4), at = (along_j ? j0 : i0) + (threadIdx.x & 15) * 4;
    mu_u<true, 4>(a.beta, a.rest, a.nesterov, it, mat, along_j, [=](int r) { return line + 16 * r; }, at, u);
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

// The operations of an iteration, in their order:
//   gram()   A = X X^T
//   poly()   B = b A + c A^2
//   apply()  X <- a X + B X
template <typename V> __host__ __device__ inline void mu_walk(int steps, V &v)
{
    for (int k = 0; k < steps; ++k) {
        v.gram();
        v.poly();
        v.apply(k + 1 == steps);
    }
}

// Writes the factors of every operation: of the old entry, and of the sum of products.  Scales are powers of two, from bounds on
// the largest singular values.
#define MU_SLACK (1.0 + 1.0 / 512.0) // for the roundings on the way: the bounds hold for exact factors
struct mu_chain {
    double a, b, c, r, sx, ra = 0.0, sa = 0.0, sb = 0.0;
    float *t;
    static constexpr double slack = MU_SLACK;
    __host__ __device__ mu_chain(double a_, double b_, double c_, double r_, float *t_) : a(a_), b(b_), c(c_), r(r_ * slack), t(t_) { sx = mu_scale(r); }
    __host__ __device__ void put(double k0, double k1)
    {
        t[0] = (float)k0, t[1] = (float)k1;
        t += MU_COEF;
    }
    __host__ __device__ void gram()
    {
        ra = r * r * slack, sa = mu_scale(ra);
        put(0.0, sa / (sx * sx));
    }
    __host__ __device__ void poly()
    {
        double m = fabs(b * ra + c * ra * ra); // max |b t + c t^2| over [0, ra]
        if (c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < ra) m = fmax(m, fabs(b * b / (4.0 * c)));
        sb = mu_scale(m * slack);
        put(b * (sb / sa), c * (sb / sa) / sa);
    }
    __host__ __device__ void apply(bool last)
    {
        r = mu_largest_odd(a, b, c, r) * slack;
        const double s = last ? 1.0 : mu_scale(r);
        put(a * (s / sx), s / sb / sx);
        sx = s;
    }
};

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
    if (threadIdx.x) return;
    const mu_norm n = mu_start(red[0] + red[1] + red[2] + red[3], a.eps);
    double scale = a.sx;
    if (n.r != 1.0) {
        mu_chain chain(a.a, a.b, a.c, n.r, a.table + (size_t)blockIdx.x * a.steps * MU_OPS * MU_COEF);
        scale = chain.sx;
        mu_walk(a.steps, chain);
    }
    a.x0[2 * blockIdx.x] = n.x0 * scale;
    a.x0[2 * blockIdx.x + 1] = n.r == 1.0 ? 1.0 : 0.0;
}

// hi = fp16(v), lo = fp16(v - hi), in two instructions an entry: pairs are converted together, and the difference takes hi as
// it is (v_fma_mix_f32; minus_one is hidden from the compiler, which would turn the product into conversions and subtractions).
template <int N> __device__ __forceinline__ void mu_split(const float (&v)[N], mu_h (&hi)[N], mu_h (&lo)[N])
{
    typedef mu_h h2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    float minus_one = -1.0f;
    asm("" : "+s"(minus_one));
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const h2 h = __builtin_convertvector((f2){v[e], v[e + 1]}, h2);
        const h2 l = __builtin_convertvector((f2){__builtin_fmaf((float)h[0], minus_one, v[e]), __builtin_fmaf((float)h[1], minus_one, v[e + 1])}, h2);
        hi[e] = h[0], hi[e + 1] = h[1], lo[e] = l[0], lo[e + 1] = l[1];
    }
}
__device__ __forceinline__ void mu_split4(float v0, float v1, float v2, float v3, mu_h4 &hi, mu_h4 &lo)
{
    const float v[4] = {v0, v1, v2, v3};
    mu_h h[4], l[4];
    mu_split<4>(v, h, l);
    hi = mu_h4{h[0], h[1], h[2], h[3]}, lo = mu_h4{l[0], l[1], l[2], l[3]};
}
__device__ __forceinline__ void mu_split8(const float (&v)[8], mu_h8 &hi, mu_h8 &lo)
{
    mu_h h[8], l[8];
    mu_split<8>(v, h, l);
    hi = mu_h8{h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[7]}, lo = mu_h8{l[0], l[1], l[2], l[3], l[4], l[5], l[6], l[7]};
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
    const mu_factor scale(a.x0[2 * (it.first + mat)]);
    float u[16];
    const int first = threadIdx.x >> 4, x = (threadIdx.x & 15) * 4, line = (along_j ? i0 : j0) + first;
    mu_u<false, 4>(a.beta, a.rest, a.nesterov, it, mat, along_j, [=](int r) { return line + 16 * r; }, (along_j ? j0 : i0) + x, u);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = along_j ? first + 16 * r : x + e, j = along_j ? x + e : first + 16 * r;
            tile[i][j] = i0 + i < it.n && j0 + j < it.l ? scale * u[4 * r + e] : 0.0f; // (the scale may be NaN)
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
        for (int q = 0; q < 8; ++q) v[q] = tile[row][c + q];
        mu_split8(v, hi, lo);
        __builtin_memcpy(w.x32 + (size_t)(i0 + row) * it.lp + j0 + c, v, 32);
        *(mu_h8 *)(w.x + at) = hi;
        *(mu_h8 *)(w.x + at + 32) = lo;
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = tile[c + q][row];
        mu_split8(v, hi, lo);
        *(mu_h8 *)(w.xt + at_t) = hi;
        *(mu_h8 *)(w.xt + at_t + 32) = lo;
    }
}

enum { MU_GRAM = 0, MU_SYM = 1, MU_APPLY = 2, MU_LAST = 3 };

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
//   MU_GRAM: A = k1 sum      MU_SYM: B = k0 A + k1 sum      MU_APPLY: X = k0 X + k1 sum; MU_LAST: p
#define MU_PITCH(NI) (32 * (NI) + 4)
// The factors of an operation.  What is loaded for them is asked for before the products and looked at behind them.
struct mu_factors {
    const mu_args &a;
    double ready; // not 0: the launch's own factors hold
    float t0, t1;
    __device__ __forceinline__ mu_factors(const mu_args &args, int matrix) : a(args)
    {
        const float *t = a.table + ((size_t)matrix * a.steps * MU_OPS + a.op) * MU_COEF;
        ready = a.x0[2 * matrix + 1], t0 = t[0], t1 = t[1];
    }
    __device__ __forceinline__ float k0() const { return ready != 0.0 ? a.k[0] : t0; }
    __device__ __forceinline__ float k1() const { return ready != 0.0 ? a.k[1] : t1; }
};

// The old entries in float32 that a lane combines with its part of a strip of 32 x 32, asked for before the products: a launch of
// a few 64-tiles takes 9.0 us, 9.9 where they are asked for behind them.
struct mu_early {
    float4 o[4];
};
template <int MODE, int NI, bool EARLY>
__device__ __forceinline__ void mu_strip(const mu_factors &f, const mu_item &it, int mat, const mu_mat &w,
                                         const mu_f16 (&acc)[NI], int i0, int j0, bool mirror, float *lds, int lane, const mu_early &early)
{
    constexpr int PITCH = MU_PITCH(NI), LANES = 8 * NI, ROWS = 64 / LANES; // lanes of a row, rows of a turn
    const int ld = MODE >= MU_APPLY ? it.lp : it.np;
    const float *old = MODE >= MU_APPLY ? w.x32 : w.a32;
    float *full = MODE == MU_APPLY ? w.x32 : w.a32; // (MU_GRAM; B is a factor only)
    mu_h *out = MODE == MU_APPLY ? w.x2 : MODE == MU_GRAM ? w.a : w.b, *out_t = MODE == MU_APPLY ? w.xt2 : out;
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
    const float k0 = f.k0(), k1 = f.k1();
#pragma unroll(MODE == MU_LAST ? 1 : 4)
    for (int turn = 0; turn < 32 / ROWS; ++turn) {
        const int r = turn * ROWS + lane / LANES, c = (lane % LANES) * 4, i = i0 + r, j = j0 + c;
        if (i >= it.np || j >= ld) continue;
        float4 v = *(const float4 *)(lds + r * PITCH + c);
        const float4 o = EARLY ? early.o[turn & 3] : MODE == MU_GRAM ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *(const float4 *)(old + (size_t)i * ld + j);
        v = make_float4(k0 * o.x + k1 * v.x, k0 * o.y + k1 * v.y, k0 * o.z + k1 * v.z, k0 * o.w + k1 * v.w);
        if (back) *(float4 *)(lds + r * PITCH + c) = v;
        if (MODE == MU_LAST) {
            if (by_rows && i < it.n && j < it.l) mu_update4(it, mat * it.ps[0] + i * it.ps[1] + j * it.ps[2], it.ps[2], min(4, it.l - j), v);
        } else {
            mu_h4 hi, lo;
            mu_split4(v.x, v.y, v.z, v.w, hi, lo);
            if (MODE == MU_GRAM || MODE == MU_APPLY) *(float4 *)(full + (size_t)i * ld + j) = v;
            *(mu_h4 *)(out + mu_at(i, j, ld)) = hi;
            *(mu_h4 *)(out + mu_at(i, j, ld) + 32) = lo;
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
            mu_split8(v, hi, lo);
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

// Neighbouring workgroups go to different XCDs: each of the eight takes a run of neighbouring ones of the n (-1: none is left).
__host__ __device__ inline int mu_by_xcd(int xcd, int rank, int n)
{
    const int first = (int)((long long)n * xcd / 8), end = (int)((long long)n * (xcd + 1) / 8);
    return first + rank < end ? first + rank : -1;
}

// One tile of a product.  LDS holds two stages of 32 k: T rows of P and T of Q, 128 bytes each; the eight 16-byte chunks of a
// row (four of hi, four of lo) lie at chunk ^ ((row >> 1) & 7), which spreads the 16 rows that a quarter wave reads over all
// 64 banks.  The loads go from global memory to LDS directly, one stage ahead of the products (three for the smallest tile).
// Bound: the matrix cores for the 256-tile (B X of 4096 x 4096: 352 us = 1.17 PFLOP/s; the chip lowers its clock under this
// load: on zeros the whole call takes 2.9 ms, on numbers 3.9).  The 128-tile reaches 0.85 to 0.95 (four symmetric products of 2048:
// 115 to 121 us): it reads LDS twice as often for a product and has its loads only one shorter stage ahead.  Eight waves of 64 x 32 hide
// that better than four of 64 x 64 (a layer's four weights, when blocks of steps were taken, 3.10 against 3.19 ms; two of 128 x 64:
// 3.38; eight with four stages: 3.27).  The 64-tile is bound by its loads (eight symmetric products of 1024: 47 us).
template <int T, int WM, int WN, int MODE>
__global__ __launch_bounds__(64 * WM * WN) void mu_product_kernel(mu_args a)
{
    constexpr int WAVES = WM * WN, MI = T / WM / 32, NI = T / WN / 32;
    // the smallest tile's products of a stage take less time than its loads: its loads run three stages ahead
    constexpr int STAGES = T == 64 ? 4 : 2;
    __shared__ __attribute__((aligned(1024))) char buf0[4 * T * 64];
    __shared__ __attribute__((aligned(1024))) char buf1[4 * T * 64];
    __shared__ __attribute__((aligned(1024))) char buf2[STAGES > 2 ? 4 * T * 64 : 1024];
    __shared__ __attribute__((aligned(1024))) char buf3[STAGES > 2 ? 4 * T * 64 : 1024];
    // First the workgroups of the whole tiles, item by item, an eighth of each item on every XCD (the items' k differ); then
    // those of the tiles that are cut along k.
    int rank = blockIdx.x >> 3, tile = -1, k = 0;
    for (; k < a.n_items && tile < 0; ++k) {
        const int n = min(a.start[k + 1], a.direct) - a.start[k], each = (n + 7) / 8;
        if (n <= 0) continue;
        if (rank < each) {
            tile = mu_by_xcd((blockIdx.x + a.start[k]) & 7, rank, n); // (so that items of a few tiles do not all take the same XCDs)
            if (tile < 0) return;
            tile += a.start[k--];
        } else {
            rank -= each;
        }
    }
    const int units_all = (a.start[a.n_items] - a.direct) * a.splits;
    const bool part = tile < 0;
    const int unit = part ? mu_by_xcd(blockIdx.x & 7, rank, units_all) : 0;
    if (unit < 0) return;
    if (part) {
        tile = a.direct + unit / a.splits;
        k = mu_find(a, tile);
    }
    const mu_item &it = a.it[k];
    const int ti = (it.np + T - 1) / T, tj = MODE >= MU_APPLY ? (it.lp + T - 1) / T : ti;
    const int per = MODE >= MU_APPLY ? ti * tj : ti * (ti + 1) / 2, local = tile - a.start[k];
    const int mat = local / per;
    int i0, j0;
    mu_place<MODE>(local % per, ti, tj, i0, j0);
    i0 *= T, j0 *= T;
    const mu_mat w = mu_planes(a, it, mat);
    const mu_factors factors(a, it.first + mat);
    const int K = MODE == MU_GRAM ? it.lp : it.np, jrows = MODE >= MU_APPLY ? it.lp : it.np;
    const mu_h *P = MODE == MU_GRAM ? w.x : MODE == MU_SYM ? w.a : w.b, *Q = MODE == MU_GRAM ? w.x : MODE == MU_SYM ? w.a : w.xt;
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

    constexpr bool EARLY = T == 64 && (MODE == MU_SYM || MODE == MU_APPLY);
    mu_early early;
    if (EARLY) { // (rows and columns of a 64-tile all lie inside)
        const float *old = MODE == MU_APPLY ? w.x32 : w.a32;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            early.o[q] = *(const float4 *)(old + (size_t)(i0 + wi * 32 + lane / 8 + 8 * q) * (MODE == MU_APPLY ? it.lp : it.np) + j0 + wj * 32 + lane % 8 * 4);
    }
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
        // lgkmcnt(0): this stage is read; vmcnt: of the loads those of the next stage have arrived
        __builtin_amdgcn_s_waitcnt(0x0070 | (STAGES - 2) * 2 * FILLS);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        stage(buf, min(k0 + STAGES * MU_BK, k_end - MU_BK));
        read(f0, next, 0);
        products(f1);
    };
    static_assert((STAGES - 1) * 2 * FILLS < 16 || STAGES == 2, "");
    int k0 = k_first;
    auto begin = [&](char *first, char *second, char *third, char *fourth) {
        stage(first, k0);
        stage(second, k0 + MU_BK);
        if (STAGES > 2) {
            stage(third, min(k0 + 2 * MU_BK, k_end - MU_BK));
            stage(fourth, min(k0 + 3 * MU_BK, k_end - MU_BK));
        }
        __builtin_amdgcn_s_waitcnt(STAGES > 2 ? 0x0F70 | (STAGES - 1) * 2 * FILLS : 0x0F70); // the first stage is there
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        read(f0, first, 0);
    };
    if (STAGES == 2) {
        begin(buf0, buf1, buf2, buf3);
        for (; k0 < k_end; k0 += 2 * MU_BK) {
            turn(buf0, buf1, k0);
            turn(buf1, buf0, k0 + MU_BK);
        }
    } else {
        if ((k_end - k0) & (2 * MU_BK)) { // two stages first, so that four remain a turn
            begin(buf2, buf3, buf0, buf1);
            turn(buf2, buf3, k0);
            turn(buf3, buf0, k0 + MU_BK);
            k0 += 2 * MU_BK;
        } else {
            begin(buf0, buf1, buf2, buf3);
        }
        for (; k0 < k_end; k0 += 4 * MU_BK) {
            turn(buf0, buf1, k0);
            turn(buf1, buf2, k0 + MU_BK);
            turn(buf2, buf3, k0 + 2 * MU_BK);
            turn(buf3, buf0, k0 + 3 * MU_BK);
        }
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
        mu_strip<MODE, NI, EARLY>(factors, it, mat, w, acc[x], i0 + (wi * MI + x) * 32, j0 + wj * NI * 32, mirror, lds, lane, early);
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
    const int per = MODE >= MU_APPLY ? ti * tj : ti * (ti + 1) / 2, local = tile - a.start[k];
    const int mat = local / per;
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
    const mu_factors factors(a, it.first + mat);
    mu_strip<MODE, NI, false>(factors, it, mat, w, acc, i0 + (wi * MI + x) * 32, j0 + wj * NI * 32, MODE == MU_APPLY || i0 != j0, lds, lane,
                              mu_early());
}

// A matrix that fits one workgroup's LDS (128 x 208, 96 x 320, 64 x 512, 32 x 1,024 and less) goes through all its steps there, in one
// launch: X as rows of hi then lo, and A, then B, as rows of hi then lo; rows are 16 bytes longer than their entries, so that
// 16 of them start in different banks.  Each wave keeps its 32 x 32 tiles of X, and of A on and above the diagonal, in float32
// in registers from step to step.  X^T for B X is read from X by the transposing LDS read: of 16 lanes that address four
// rows of 16 entries it gives each lane a column's four.
// Bound: the matrix cores of one CU and the barriers (five a step).
#define MU_SMALL_WAVES 16
#define MU_SMALL_LDS (158 * 1024) // of 160 KB; the static arrays take the rest
#define MU_SMALL_TILES 2          // of X for a wave at most

__host__ __device__ inline int mu_small_n(int n) { return (n + 31) / 32 * 32; }
__host__ __device__ inline int mu_small_l(int l) { return (l + 15) / 16 * 16; }
// A symmetric matrix of nt x nt blocks of 32 x 32 is kept as its blocks on and above the diagonal, row by row; what lies below is
// read from above it, by columns.  A block: rows of 32 hi, 32 lo and 16 bytes.
#define MU_BLOCK_ROW 144
#define MU_BLOCK (32 * MU_BLOCK_ROW)
__host__ __device__ inline int mu_block(int ti, int tj, int nt) { return (ti * nt - ti * (ti - 1) / 2 + tj - ti) * MU_BLOCK; }
// Bytes of a row of X.  A direct read takes 16 bytes each from 16 rows: of all 64 banks once if the pitch is an odd number of 16
// bytes; a read by columns 64 each from four rows: twice, if that number is not 1 from a multiple of 16 (else four times).
__host__ __device__ inline int mu_small_pitch(int lp) { return 4 * lp + (lp % 64 ? 16 : 48); }
static inline int mu_small_bytes(int n, int l) // 0: too large
{
    const long long np = mu_small_n(n), lp = mu_small_l(l), bytes = np * mu_small_pitch((int)lp) + mu_block((int)np / 32, (int)np / 32, (int)np / 32);
    return np <= 128 && bytes <= MU_SMALL_LDS && (lp + 31) / 32 <= MU_SMALL_TILES * (MU_SMALL_WAVES / (np / 32)) ? (int)bytes : 0;
}

__device__ __forceinline__ mu_h4 mu_read_column(const char *p)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(mu_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
}

// hi and lo of four neighbouring entries
__device__ __forceinline__ void mu_put4(char *hi_at, char *lo_at, float v0, float v1, float v2, float v3)
{
    mu_h4 hi, lo;
    mu_split4(v0, v1, v2, v3, hi, lo);
    *(mu_h4 *)hi_at = hi;
    *(mu_h4 *)lo_at = lo;
}

__device__ __forceinline__ void mu_put_block(char *block, int lane, const mu_f16 &v)
{
    char *const at = block + (lane & 31) * MU_BLOCK_ROW + 8 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) mu_put4(at + 16 * q, at + 16 * q + 64, v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

struct mu_pair {
    mu_h8 hi, lo;
};
// A lane's eight k of a row that lies in LDS as it is.  p: the row at its first k.
__device__ __forceinline__ mu_pair mu_by_row(const char *p, int lo) { return {*(const mu_h8 *)p, *(const mu_h8 *)(p + lo)}; }
// ... of a column of what lies there.  p: where mu_column_at says, in the row of the first k.
__device__ __forceinline__ mu_pair mu_by_column(const char *p, int pitch, int lo)
{
    const mu_h4 h0 = mu_read_column(p), h1 = mu_read_column(p + 4 * pitch), l0 = mu_read_column(p + lo), l1 = mu_read_column(p + 4 * pitch + lo);
    return {__builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7)};
}
// of 16 lanes four address the same row k, 16 columns; the upper half of a wave takes k from 8 on
__device__ __forceinline__ int mu_column_at(int lane, int pitch) { return (8 * (lane >> 5) + (lane & 15) / 4) * pitch + 32 * (lane >> 4 & 1) + 8 * (lane & 3); }

__device__ __forceinline__ void mu_three(const mu_pair &p, const mu_pair &q, mu_f16 &acc)
{
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.lo, p.hi, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.hi, p.lo, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.hi, p.hi, acc, 0, 0, 0);
}
// the first of a sum: 0 as an operand of the instruction instead of 16 registers that are cleared
__device__ __forceinline__ mu_f16 mu_three(const mu_pair &p, const mu_pair &q)
{
    mu_f16 acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.lo, p.hi, (mu_f16)(0.0f), 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.hi, p.lo, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(q.hi, p.hi, acc, 0, 0, 0);
}
__device__ __forceinline__ void mu_zero(mu_f16 &acc)
{
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
}

__global__ __launch_bounds__(64 * MU_SMALL_WAVES) void mu_small_kernel(mu_args by_value)
{
    // The arguments where they lie (the first one starts the kernel's argument segment): with this many uses of `by_value` the
    // compiler copies all 3.5 KB of it to every thread's scratch.
    const mu_args &a = *(const mu_args *)__builtin_amdgcn_kernarg_segment_ptr();
    extern __shared__ __attribute__((aligned(16))) char mu_lds[];
    __shared__ double red[MU_SMALL_WAVES];
    __shared__ float own[MU_STEPS * MU_OPS * MU_COEF];
    int k = 0;
    while (k + 1 < a.n_items && (int)blockIdx.x >= a.it[k + 1].first) ++k;
    const mu_item &it = a.it[k];
    const int mat = blockIdx.x - it.first, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 31, half = lane >> 5; // of a fragment: its row, and which 8 of 16 k
    const int np = mu_small_n(it.n), lp = mu_small_l(it.l), nt = np / 32;
    const int px = mu_small_pitch(lp);
    char *const X = mu_lds, *const A = mu_lds + np * px;

    // A wave's tiles of X all lie in the same 32 rows (they share what they read of B): tiles (xi, xj + t groups).
    const int groups = MU_SMALL_WAVES / nt, xi = wave % nt, xj = wave / nt, last = wave < groups * nt ? (lp + 31) / 32 : 0;
    // A tile is held as four neighbouring columns in every four registers.  They are read (and at the end written) in pieces of
    // four along the side on which g (p) is contiguous, and change hands through LDS, where X will be.
    double s = 0.0;
    const bool along_j = it.gs[2] == 1 || it.gs[1] != 1;
#pragma unroll 1
    for (int tile = xj; tile < last; tile += groups) {
        const int i0 = xi * 32, j0 = tile * 32, x = lane % 8 * 4, line = (along_j ? i0 : j0) + lane / 8;
        float u[16];
        mu_u<true, 4>(a.beta, a.rest, a.nesterov, it, mat, along_j, [=](int r) { return line + 8 * r; }, (along_j ? j0 : i0) + x, u);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + (along_j ? 8 * r + lane / 8 : x), j = j0 + (along_j ? x : 8 * r + lane / 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) s += (double)u[4 * r + e] * u[4 * r + e];
            if (j >= lp) continue; // (a piece lies within lp or outside)
            if (along_j) {
                *(float4 *)(X + i * px + 4 * j) = make_float4(u[4 * r], u[4 * r + 1], u[4 * r + 2], u[4 * r + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) *(float *)(X + (i + e) * px + 4 * j) = u[4 * r + e];
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
        if ((int)threadIdx.x < a.steps * MU_OPS * MU_COEF) own[threadIdx.x] = a.std[threadIdx.x];
        x0 *= a.sx;
    } else { // a norm below eps
        lrb_barrier(); // red has been read
        if (threadIdx.x == 0) {
            mu_chain chain(a.a, a.b, a.c, n.r, own);
            red[0] = chain.sx;
            mu_walk(a.steps, chain);
        }
        lrb_barrier();
        x0 *= red[0];
    }
    const mu_factor scale(x0);
    const float *coef = own;
    float x[MU_SMALL_TILES][16];
#pragma unroll
    for (int t = 0; t < MU_SMALL_TILES; ++t) {
        const int tile = xj + t * groups;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = xi * 32 + row, j = tile * 32 + 4 * half + 8 * q;
            const float4 v = tile < last && j < lp ? *(const float4 *)(X + i * px + 4 * j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            x[t][4 * q] = scale * v.x, x[t][4 * q + 1] = scale * v.y, x[t][4 * q + 2] = scale * v.z, x[t][4 * q + 3] = scale * v.w;
        }
    }

    lrb_barrier(); // all have read: what follows writes hi and lo there
    // the wave's tile of the symmetric products, on or above the diagonal
    int ti = 0, tj = wave;
    while (ti < nt && tj >= nt - ti) tj -= nt - ti++;
    tj += ti;
    const bool sym = ti < nt;
    for (int step = 0; step < a.steps; ++step, coef += MU_OPS * MU_COEF) {
        // the addresses below are made anew in every step: kept over the steps, all of them together spill
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int row = lane & 31, half = lane >> 5;
#pragma unroll
        for (int t = 0; t < MU_SMALL_TILES; ++t) {
            const int tile = xj + t * groups, i = xi * 32 + row, j = tile * 32 + 4 * half;
            if (tile >= last) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (j + 8 * q >= lp) continue;
                char *const at = X + i * px + 2 * (j + 8 * q);
                mu_put4(at, at + 2 * lp, x[t][4 * q], x[t][4 * q + 1], x[t][4 * q + 2], x[t][4 * q + 3]);
            }
        }
        lrb_barrier();
        mu_f16 full, acc;
        mu_zero(full);
        if (sym) {
            const char *p = X + (ti * 32 + row) * px + 16 * half, *q = X + (tj * 32 + row) * px + 16 * half;
            if (ti == tj) {
                const mu_pair f = mu_by_row(p, 2 * lp);
                full = mu_three(f, f);
#pragma unroll 2
                for (int k0 = 16; k0 < lp; k0 += 16) {
                    const mu_pair v = mu_by_row(p += 32, 2 * lp);
                    mu_three(v, v, full);
                }
            } else {
                full = mu_three(mu_by_row(p, 2 * lp), mu_by_row(q, 2 * lp));
#pragma unroll 2
                for (int k0 = 16; k0 < lp; k0 += 16) mu_three(mu_by_row(p += 32, 2 * lp), mu_by_row(q += 32, 2 * lp), full);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) full[e] *= coef[1];
            mu_put_block(A + mu_block(ti, tj, nt), lane, full);
        }
        lrb_barrier();
        const int by_row = row * MU_BLOCK_ROW + 16 * half, by_column = mu_column_at(lane, MU_BLOCK_ROW);
        mu_zero(acc);
        if (sym) {
            for (int kb = 0; kb < ti; ++kb) {
                const char *p = A + mu_block(kb, ti, nt) + by_column, *q = A + mu_block(kb, tj, nt) + by_column;
#pragma unroll
                for (int h = 0; h < 2; ++h, p += 16 * MU_BLOCK_ROW, q += 16 * MU_BLOCK_ROW)
                    mu_three(mu_by_column(p, MU_BLOCK_ROW, 64), mu_by_column(q, MU_BLOCK_ROW, 64), acc);
            }
            for (int kb = ti; kb < tj; ++kb) {
                const char *p = A + mu_block(ti, kb, nt) + by_row, *q = A + mu_block(kb, tj, nt) + by_column;
#pragma unroll
                for (int h = 0; h < 2; ++h, p += 32, q += 16 * MU_BLOCK_ROW) mu_three(mu_by_row(p, 64), mu_by_column(q, MU_BLOCK_ROW, 64), acc);
            }
            for (int kb = tj; kb < nt; ++kb) {
                const char *p = A + mu_block(ti, kb, nt) + by_row, *q = A + mu_block(tj, kb, nt) + by_row;
#pragma unroll
                for (int h = 0; h < 2; ++h, p += 32, q += 32) mu_three(mu_by_row(p, 64), mu_by_row(q, 64), acc);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = coef[2] * full[e] + coef[3] * acc[e];
        }
        lrb_barrier();
        if (sym) mu_put_block(A + mu_block(ti, tj, nt), lane, acc);
        lrb_barrier();
        if (xj < last) { // both tiles at once
            static_assert(MU_SMALL_TILES == 2, "");
            const bool two = xj + groups < last;
            mu_f16 other;
            mu_zero(acc), mu_zero(other);
            // rows k of X, read by columns; columns past the end give what is not kept
            const char *q = X + mu_column_at(lane, px) + 64 * xj;
            for (int kb = 0; kb < nt; ++kb) {
                const char *p = A + (kb < xi ? mu_block(kb, xi, nt) + by_column : mu_block(xi, kb, nt) + by_row);
#pragma unroll
                for (int h = 0; h < 2; ++h, q += 16 * px) {
                    const mu_pair v = kb < xi ? mu_by_column(p + h * 16 * MU_BLOCK_ROW, MU_BLOCK_ROW, 64) : mu_by_row(p + h * 32, 64);
                    mu_three(v, mu_by_column(q, px, 2 * lp), acc);
                    if (two) mu_three(v, mu_by_column(q + 64 * groups, px, 2 * lp), other);
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[0][e] = coef[4] * x[0][e] + coef[5] * acc[e];
                x[1][e] = coef[4] * x[1][e] + coef[5] * other[e];
            }
        }
        lrb_barrier();
    }
#pragma unroll
    for (int t = 0; t < MU_SMALL_TILES; ++t) {
        const int tile = xj + t * groups;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = xi * 32 + row, j = tile * 32 + 4 * half + 8 * q;
            if (tile < last && j < lp) *(float4 *)(X + i * px + 4 * j) = make_float4(x[t][4 * q], x[t][4 * q + 1], x[t][4 * q + 2], x[t][4 * q + 3]);
        }
    }
    mu_wave_sync();
    const bool by_rows = it.ps[2] == 1 || it.ps[1] != 1;
#pragma unroll 1
    for (int tile = xj; tile < last; tile += groups) {
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
            const int line = 8 * q + lane / 8, at = lane % 8 * 4;
            const int i = xi * 32 + (by_rows ? line : at), j = tile * 32 + (by_rows ? at : line);
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

// The tile: the largest that still fills most of the chip (a larger tile loads less for each product): 256 CUs take one each of
// 256, two each of 128.  (Eight symmetric products of 1024: 288 tiles of 128 and 1088 of 64 both take 47 us.)  Both symmetric products take the same (A's
// float32 is there on and above the diagonal's tiles only).
// The cut: a round of 256 tiles gives every CU one; the tiles that are left over behind the last whole round are cut along k so
// that all CUs share them, if that saves more than the launch that joins the parts takes (about 5 us: 14 units of 64 k of the
// smallest tile, five of the middle one, two of the largest).  4096 x 4096, symmetric product of 528 tiles: 302 us whole, 231 +
// 12 with the last 16 cut (193 + 9 since a tile has eight waves).
static mu_plan mu_lay_out(const mu_args &a, int mode)
{
    const bool symmetric = mode <= MU_SYM;
    mu_plan p;
    p.T = mu_tiles(a, symmetric, 256, nullptr) >= 200 ? 256 : mu_tiles(a, symmetric, 128, nullptr) >= 400 ? 128 : 64;
    p.tiles = mu_tiles(a, symmetric, p.T, nullptr);
    const long long rest = p.tiles % 256;
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
    long long s = 256 / rest;
    if (s > units / 3) s = units / 3; // at least 192 k a part
    if (s < 2 || units - units / s < (p.T == 64 ? 14 : p.T == 128 ? 5 : 2)) return p;
    p.direct = (int)(p.tiles - rest), p.splits = (int)s;
    return p;
}

template <int T, int WM, int WN, int MODE> static void mu_launch_tiles(const mu_args &a, const mu_plan &p, hipStream_t st)
{
    const long long cut = p.tiles - p.direct, units = cut * p.splits;
    long long grid = (units + 7) / 8;
    for (int k = 0; k < a.n_items; ++k) {
        const int n = (a.start[k + 1] < p.direct ? a.start[k + 1] : p.direct) - a.start[k];
        if (n > 0) grid += (n + 7) / 8;
    }
    hipLaunchKernelGGL((mu_product_kernel<T, WM, WN, MODE>), dim3((unsigned)(grid * 8)), dim3(64 * WM * WN), 0, st, a);
    if (cut) hipLaunchKernelGGL((mu_join_kernel<T, WM, WN, MODE>), dim3((unsigned)(cut * (T / 32) * WN)), dim3(64), 0, st, a);
}

template <int MODE> static void mu_launch_product(mu_args &a, hipStream_t st)
{
    const mu_plan p = mu_lay_out(a, MODE);
    mu_tiles(a, MODE <= MU_SYM, p.T, a.start);
    a.direct = p.direct, a.splits = p.splits;
    if (p.T == 256) mu_launch_tiles<256, 2, 4, MODE>(a, p, st);
    else if (p.T == 128) mu_launch_tiles<128, 2, 4, MODE>(a, p, st);
    else mu_launch_tiles<64, 2, 2, MODE>(a, p, st);
}

// Launches the operations of an iteration.
struct mu_launcher {
    mu_args &g;
    hipStream_t st;
    template <int MODE> void launch()
    {
        memcpy(g.k, g.std + g.op * MU_COEF, sizeof(g.k));
        mu_launch_product<MODE>(g, st);
        ++g.op;
    }
    void gram() { launch<MU_GRAM>(); }
    void poly() { launch<MU_SYM>(); }
    void apply(bool last)
    {
        if (last) launch<MU_LAST>();
        else launch<MU_APPLY>();
        g.flip ^= 1;
    }
};

// A run of items (or of some matrices of one) that fits the descriptors and MU_WS_MOST bytes, and what it takes.
#define MU_WS_MOST (4ull << 30)
#define MU_MATS_MOST 4096
struct mu_group {
    mu_args a;
    int lds; // of a group whose matrices fit a workgroup's LDS: the most that one takes; else 0
    int mats;
    long long tiles;
    uint64_t planes;
    // sizes of what lies behind the planes
    uint64_t x0_bytes() const { return ((uint64_t)mats * 16 + 255) / 256 * 256; }
    uint64_t sums_bytes() const { return ((uint64_t)tiles * 8 + 255) / 256 * 256; }
    uint64_t table_bytes() const { return ((uint64_t)mats * MU_STEPS * MU_OPS * MU_COEF * 4 + 255) / 256 * 256; }
    uint64_t bytes() const
    {
        if (lds) return 0;
        uint64_t parts = 0;
        for (int mode = MU_GRAM; mode <= MU_LAST; ++mode) {
            const uint64_t b = mu_lay_out(a, mode).part_bytes();
            parts = b > parts ? b : parts;
        }
        return planes + parts + x0_bytes() + sums_bytes() + table_bytes();
    }
};

// Calls `go(group)` for each group of the list in turn, those of small matrices first; stops at its first non-zero answer.
template <typename F> static int mu_each_group(const lrb_muon_item *items, int n_items, F go)
{
    // the largest first: what is left for the last, unfilled round of a launch are then the least
    std::vector<int> order(n_items);
    for (int k = 0; k < n_items; ++k) order[k] = k;
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return items[x].rows * items[x].cols > items[y].rows * items[y].cols; });
    for (int small = 1; small >= 0; --small) {
        mu_group gr = {};
        for (int k : order) {
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
        // sides up to 2^22 and planes below 2^31 entries, both sides padded to 64: the kernels' 32-bit indices hold
        if (s.rows > (1 << 22) || s.cols > (1 << 22) || (s.rows + 63) / 64 * 64 * ((s.cols + 63) / 64 * 64) > INT_MAX) return false;
        if (!s.p || !s.g || s.p_type < LRB_F32 || s.p_type > LRB_F16 || s.g_type < LRB_F32 || s.g_type > LRB_F16) return false;
        if (s.m && (s.m_type < LRB_F32 || s.m_type > LRB_F16)) return false;
    }
    return true;
}

static double mu_bound(int steps, double a, double b, double c, double slack)
{
    double r = slack, most = 1.0;
    for (int k = 0; k < steps && k < MU_STEPS && r <= 1e9; ++k) {
        r = mu_largest_odd(a, b, c, r) * slack;
        most = most >= r ? most : r; // a NaN stays
    }
    return most;
}

// Where the exact bound is small, but the one with the slack that the factors' scales are made from is not (x^5 keeps 1 where it
// is, and takes what is beyond it away), a rounding could grow as the latter says, and the scales would leave nothing of a 16-bit
// factor: then the latter is the answer.
extern "C" double lrb_muon_bound(int steps, float a, float b, float c)
{
    const double exact = mu_bound(steps, a, b, c, 1.0), slack = mu_bound(steps, a, b, c, MU_SLACK);
    return exact <= LRB_MUON_DIVERGED && !(slack <= LRB_MUON_DIVERGED) ? slack : exact;
}

extern "C" uint64_t lrb_muon_ws_bytes(const lrb_muon_item *items, int n_items)
{
    if (n_items <= 0 || !items || !mu_items_fit(items, n_items)) return 0;
    uint64_t most = 0;
    try {
        mu_each_group(items, n_items, [&](mu_group &gr) {
            if (gr.bytes() > most) most = gr.bytes();
            return LRB_OK;
        });
    } catch (const std::bad_alloc &) {
        return UINT64_MAX; // no workspace is as large: the call that follows is refused
    }
    return most;
}

extern "C" int lrb_muon_dev(int device, void *stream, const lrb_muon_item *items, int n_items, double momentum, int nesterov, int steps,
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
    float std[MU_STEPS * MU_OPS * MU_COEF] = {};
    mu_chain chain(a, b, c, 1.0, std);
    const double sx = chain.sx;
    mu_walk(steps, chain);
    try {
        return mu_each_group(items, n_items, [&](mu_group &gr) -> int {
            mu_args &g = gr.a;
            g.steps = steps, g.beta = (float)momentum, g.rest = (float)(1.0 - momentum), g.nesterov = nesterov, g.eps = eps, g.a = a, g.b = b, g.c = c;
            g.sx = sx;
            memcpy(g.std, std, sizeof(std));
            if (gr.lds) {
                static lrb_per_device_once raised;
                HIP_TRY(lrb_raise_lds(raised, device, (const void *)mu_small_kernel, MU_SMALL_LDS));
                hipLaunchKernelGGL(mu_small_kernel, dim3(gr.mats), dim3(64 * MU_SMALL_WAVES), gr.lds, st, g);
                HIP_TRY(hipGetLastError());
                return LRB_OK;
            }
            g.ws = (char *)d_ws;
            char *at = g.ws + gr.planes;
            g.x0 = (double *)at, at += gr.x0_bytes();
            g.part = (double *)at, at += gr.sums_bytes();
            g.table = (float *)at, at += gr.table_bytes();
            g.parts = (float *)at;
            hipLaunchKernelGGL(mu_momentum_kernel, dim3((unsigned)gr.tiles), dim3(256), 0, st, g);
            hipLaunchKernelGGL(mu_table_kernel, dim3(gr.mats), dim3(256), 0, st, g);
            hipLaunchKernelGGL(mu_split_kernel, dim3((unsigned)gr.tiles), dim3(256), 0, st, g);
            mu_launcher launcher{g, st};
            mu_walk(steps, launcher);
            HIP_TRY(hipGetLastError());
            return LRB_OK;
        });
    } catch (const std::bad_alloc &) {
        lrb_set_error("out of memory%s%s", "", "");
        return LRB_ERR_NOMEM;
    }
}
