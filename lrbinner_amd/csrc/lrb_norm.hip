// lrb_norm.hip -- K9: layer normalisation over the last axis, forward and backward, gfx950 only.
//
//   u   = x, or keep * keep_scale * leaky_relu(x)             (what follows a linear layer in a block)
//   y   = hat * w + b,  hat = (u - mean) * rstd,  rstd = 1 / sqrt(mean((u - mean)^2) + eps)
//   g   = dy * w
//   du  = rstd * (g - mean(g) - hat * mean(g * hat)),  dx = du * du/dx
//   dw  = sum over rows of dy * hat,  db = sum over rows of dy
//
// Bound: memory.  A row is read once and stays in registers between its reductions, so a forward pass moves x and y and a backward
// pass x, dy and dx.  The mean comes first, then together the sums of the differences from it and of their squares: the former
// is what rounding (of the sum, and of 1 / cols) has left out of the mean, and corrects it and the variance.  A row of equal
// elements has variance 0 and gives b, and a mean far above the deviation costs no more than the mean's last bit.  Elements are
// divided by `cols` before they are added up: the sum of a row may be beyond float32 where its mean is not.
// TPR threads take a row, each `C` chunks of 16 bytes; the same thread meets the same columns in every row it visits, so
// w and b are loaded once per thread and the weight's gradient is summed in registers: one partial row per workgroup is
// written and a second kernel adds the partial rows in a fixed order (no atomics: the same bits run after run).
// Everything between load and store is float32.
// Measured (32,768 x 4096 bfloat16): forward 97.5 us = 5.5 TB/s, backward 160 us = 5.0 TB/s and 12 us for the join (a copy: 5.1).
#include <limits.h>
#include <math.h>

#include "lrb_device.h"

#define LN_MAX_GROUPS 1024 // workgroups of a pass: four a CU; also the largest number of partial rows of dw, db

template <typename T> struct ln_vec {
    static constexpr int V = 16 / (int)sizeof(T);
};

struct ln_args {
    const void *x, *w, *b, *dy;
    const uint8_t *keep;
    void *y, *dx;
    float *mean, *rstd; // written by the forward pass where not null, read by the backward pass
    float *part;        // [groups][2][cols]
    long long x_stride, dy_stride;
    long long rows;
    int cols;
    int w_f32; // w, b (and dw, db) are float32, else of x's type
    float eps, slope, keep_scale;
};

// A thread's V elements from column `col` on.  Rows need only their element's alignment: global loads of this target take
// any address.  Where a row ends inside the V, the thread takes the row's last V instead: it then computes some elements that
// its neighbour computes too, from the same operands in the same order, and both store the same bits; only what is summed
// over the row has to leave them out (ln_chunk::own).  So no load or store is made element by element, which for rows of
// 4095 16-bit elements cost as much as the rest (a forward pass over 8191 of them: 48 us, so 25).  Rows of fewer than V
// columns (LN_TINY) go element by element.  Rows of a multiple of V columns (LN_EVEN) have no such thread and are spared the
// selections (32,768 x 4096 bfloat16 forward: 97 us, with them 114).  A thread whose columns all lie past the end reads the
// row's last V too and stores nothing: with a branch between the loads of a row the same pass takes 129 us.
enum { LN_EVEN = 0, LN_ODD = 1, LN_TINY = 2 };
struct ln_chunk {
    int at, first;  // the first column; the first of the V elements that no neighbour has (V: none)
    __device__ __forceinline__ bool own(int i) const { return i >= first; }
    __device__ __forceinline__ bool any(int V) const { return first < V; }
};
// whether element i of chunk c is the thread's alone
#define LN_OWN(c, i) (EDGE == LN_TINY ? at[c].at + (i) < cols : EDGE == LN_ODD ? at[c].own(i) : at[c].any(V))
template <int V, int EDGE> __device__ __forceinline__ ln_chunk ln_place(int col, int cols)
{
    ln_chunk c;
    if (EDGE == LN_TINY) {
        c.at = col, c.first = col < cols ? 0 : V;
    } else {
        c.at = min(col, cols - V), c.first = min(col - c.at, V);
    }
    return c;
}

template <typename T, int V, int EDGE> __device__ __forceinline__ void ln_load(const T *__restrict__ p, ln_chunk c, int cols, float (&o)[V])
{
    if (EDGE == LN_TINY) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = c.at + i < cols ? (float)p[c.at + i] : 0.0f;
    } else {
        T t[V];
        __builtin_memcpy(t, p + c.at, sizeof(t));
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (float)t[i];
    }
}

template <typename T, int V> __device__ __forceinline__ void ln_load_raw(const T *__restrict__ p, ln_chunk c, T (&o)[V])
{
    __builtin_memcpy(o, p + c.at, sizeof(o));
}

template <typename T, int V, int EDGE> __device__ __forceinline__ void ln_store(T *__restrict__ p, ln_chunk c, int cols, const float (&o)[V])
{
    if (EDGE == LN_TINY) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c.at + i < cols) p[c.at + i] = (T)o[i];
    } else if (c.any(V)) {
        T t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = (T)o[i];
        __builtin_memcpy(p + c.at, t, sizeof(t));
    }
}

template <typename T, int V, int EDGE>
__device__ __forceinline__ void ln_load_w(const void *w, int w_f32, ln_chunk c, int cols, float dflt, float (&o)[V])
{
    if (!w) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = dflt;
    } else if (w_f32) {
        ln_load<float, V, EDGE>((const float *)w, c, cols, o);
    } else {
        ln_load<T, V, EDGE>((const T *)w, c, cols, o);
    }
}

// keep_scale where an element is kept, 0 where it is dropped (its value then never enters, whatever it is)
template <int V, int EDGE>
__device__ __forceinline__ void ln_load_keep(const uint8_t *__restrict__ p, ln_chunk c, int cols, float scale, float (&o)[V])
{
    if (EDGE == LN_TINY) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = c.at + i < cols && p[c.at + i] ? scale : 0.0f;
    } else {
        uint8_t t[V];
        __builtin_memcpy(t, p + c.at, sizeof(t));
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = t[i] ? scale : 0.0f;
    }
}

// u of the block's activation; k: keep_scale or 0.  With slope 0 what is below 0 gives 0, -inf among it.
__device__ __forceinline__ float ln_act(float x, float slope, float k)
{
    const float f = x > 0.0f ? k : slope * k;
    return k == 0.0f || (f == 0.0f && x < 0.0f) ? 0.0f : x * f;
}

// The sum over the TPR threads of a row, in every one of them.  `red`: 2 x (TPR / 64) floats of the workgroup, used in turn
// (`flip`) so that one barrier a reduction is enough.
template <int TPR> __device__ __forceinline__ float ln_sum(float v, float *red, int &flip)
{
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (TPR > 64) {
        constexpr int NW = TPR / 64;
        float *r = red + flip * NW;
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        lrb_barrier();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) v += r[i];
    }
    return v;
}

// Two sums behind one barrier; `red`: 4 x (TPR / 64) floats.  (Where one sum and then two are made of every row, the one has the
// first quarter of `red` and the two its second half.)
// The lanes of a pair take one of the two sums each, so that both go through as many exchanges as one would.
template <int TPR> __device__ __forceinline__ void ln_sum2(float &v, float &w, float *red, int &flip)
{
    constexpr int W = TPR < 64 ? TPR : 64;
    const bool odd = threadIdx.x & 1;
    float mine = odd ? w : v, other = odd ? v : w;
    mine += __shfl_xor(other, 1, 64);
#pragma unroll
    for (int o = W / 2; o > 1; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if (TPR > 64) {
        constexpr int NW = TPR / 64;
        float *r = red + flip * 2 * NW;
        flip ^= 1;
        if ((threadIdx.x & 63) < 2) r[(odd ? NW : 0) + (threadIdx.x >> 6)] = mine;
        lrb_barrier();
        v = w = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            v += r[i];
            w += r[NW + i];
        }
    } else {
        other = __shfl_xor(mine, 1, 64);
        v = odd ? other : mine;
        w = odd ? mine : other;
    }
}

// 1 / deviation from the means of the differences from `mean` and of their squares; `mean` is put right.  A NaN stays one, and
// squares beyond float32 give 0.
__device__ __forceinline__ float ln_statistics(float off, float squares, float eps, float &mean)
{
    mean += off;
    const float var = squares < INFINITY ? fmaxf(squares - off * off, 0.0f) : squares;
    return 1.0f / sqrtf(var + eps);
}

template <typename T, int TPR, int C, bool ACT, int EDGE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ln_fwd_kernel(ln_args a)
{
    constexpr int V = ln_vec<T>::V, THREADS = TPR < 256 ? 256 : TPR, RPG = THREADS / TPR;
    __shared__ float red[4 * (TPR > 64 ? TPR / 64 : 1)];
    int flip = 0;
    const int lane = threadIdx.x % TPR, cols = a.cols;
    const float inv = 1.0f / (float)cols;
    ln_chunk at[C];
#pragma unroll
    for (int c = 0; c < C; ++c) at[c] = ln_place<V, EDGE>((c * TPR + lane) * V, cols);
    float w[C][V], b[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        ln_load_w<T, V, EDGE>(a.w, a.w_f32, at[c], cols, 1.0f, w[c]);
        ln_load_w<T, V, EDGE>(a.b, a.w_f32, at[c], cols, 0.0f, b[c]);
    }
    // every thread of a workgroup makes the same number of turns (the reductions hold barriers); rows past the end are
    // taken as row `rows - 1` and not written
    const long long turns = (a.rows + RPG - 1) / RPG;
    for (long long t = blockIdx.x; t < turns; t += gridDim.x) {
        long long row = t * RPG + threadIdx.x / TPR;
        const bool live = row < a.rows;
        if (!live) row = a.rows - 1;
        const T *x = (const T *)a.x + row * a.x_stride;
        float u[C][V];
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) ln_load<T, V, EDGE>(x, at[c], cols, u[c]);
        if (ACT) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float k[V];
                if (a.keep) {
                    ln_load_keep<V, EDGE>(a.keep + row * cols, at[c], cols, a.keep_scale, k);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) k[i] = a.keep_scale;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) u[c][i] = ln_act(u[c][i], a.slope, k[i]);
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) s = fmaf(LN_OWN(c, i) ? u[c][i] : 0.0f, inv, s);
        float mean = ln_sum<TPR>(s, red, flip), s2 = 0.0f;
        s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float e = LN_OWN(c, i) ? u[c][i] - mean : 0.0f;
                s = fmaf(e, inv, s);
                s2 = fmaf(e, e, s2);
            }
        ln_sum2<TPR>(s, s2, red, flip);
        const float rstd = ln_statistics(s, s2 * inv, a.eps, mean);
        if (!live) continue;
        if (a.mean && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        T *y = (T *)a.y + row * cols;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = (u[c][i] - mean) * rstd * w[c][i] + b[c][i];
            ln_store<T, V, EDGE>(y, at[c], cols, o);
        }
    }
}

template <typename T, int TPR, int C, bool ACT, int EDGE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ln_bwd_kernel(ln_args a)
{
    constexpr int V = ln_vec<T>::V, THREADS = TPR < 256 ? 256 : TPR, RPG = THREADS / TPR;
    __shared__ float red[4 * (TPR > 64 ? TPR / 64 : 1)];
    int flip = 0;
    const int lane = threadIdx.x % TPR, cols = a.cols;
    const float inv = 1.0f / (float)cols;
    ln_chunk at[C];
#pragma unroll
    for (int c = 0; c < C; ++c) at[c] = ln_place<V, EDGE>((c * TPR + lane) * V, cols);
    float w[C][V], dw[C][V], db[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        ln_load_w<T, V, EDGE>(a.w, a.w_f32, at[c], cols, 1.0f, w[c]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[c][i] = db[c][i] = 0.0f;
    }
    const long long turns = (a.rows + RPG - 1) / RPG;
    for (long long t = blockIdx.x; t < turns; t += gridDim.x) {
        long long row = t * RPG + threadIdx.x / TPR;
        const bool live = row < a.rows;
        if (!live) row = a.rows - 1;
        const T *x = (const T *)a.x + row * a.x_stride, *dy = (const T *)a.dy + row * a.dy_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        // between the two passes over a row its elements stay as hat and g, or, where a thread of 1024 has 16 of them and 128
        // registers, as they were read: two 16-bit numbers in the place of two float32
        constexpr bool RAW = TPR == 1024 && C * V == 16 && sizeof(T) == 2;
        float hat[RAW ? 1 : C][V], g[RAW ? 1 : C][V];
        T raw_x[RAW ? C : 1][V], raw_dy[RAW ? C : 1][V];
        uint32_t kept = 0, above = 0; // a bit an element: kept, and above 0
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (RAW) {
                ln_load_raw<T, V>(x, at[c], raw_x[RAW ? c : 0]);
                ln_load_raw<T, V>(dy, at[c], raw_dy[RAW ? c : 0]);
            } else {
                ln_load<T, V, EDGE>(x, at[c], cols, hat[RAW ? 0 : c]);
                ln_load<T, V, EDGE>(dy, at[c], cols, g[RAW ? 0 : c]);
            }
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float k[V];
            if (ACT) {
                if (a.keep) {
                    ln_load_keep<V, EDGE>(a.keep + row * cols, at[c], cols, a.keep_scale, k);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) k[i] = a.keep_scale;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float h = RAW ? (float)raw_x[RAW ? c : 0][i] : hat[RAW ? 0 : c][i], d = RAW ? (float)raw_dy[RAW ? c : 0][i] : g[RAW ? 0 : c][i];
                if (ACT) {
                    kept |= (uint32_t)(k[i] != 0.0f) << (c * V + i);
                    above |= (uint32_t)(h > 0.0f) << (c * V + i);
                    h = ln_act(h, a.slope, k[i]);
                }
                h = (h - mean) * rstd;
                if (live) {
                    dw[c][i] += d * h;
                    db[c][i] += d;
                }
                d *= w[c][i];
                if (!RAW) hat[RAW ? 0 : c][i] = h, g[RAW ? 0 : c][i] = d;
                s1 += LN_OWN(c, i) ? d : 0.0f;
                s2 += LN_OWN(c, i) ? d * h : 0.0f;
            }
        }
        if (!a.dx) continue;
        ln_sum2<TPR>(s1, s2, red, flip);
        s1 *= inv, s2 *= inv;
        if (!live) continue;
        T *dx = (T *)a.dx + row * cols;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float h = RAW ? ((float)raw_x[RAW ? c : 0][i] - mean) * rstd : hat[RAW ? 0 : c][i];
                const float d = RAW ? (float)raw_dy[RAW ? c : 0][i] * w[c][i] : g[RAW ? 0 : c][i];
                o[i] = (d - s1 - h * s2) * rstd;
                if (ACT)
                    o[i] = !(kept >> (c * V + i) & 1) ? 0.0f : o[i] * (above >> (c * V + i) & 1 ? a.keep_scale : a.slope * a.keep_scale);
            }
            ln_store<T, V, EDGE>(dx, at[c], cols, o);
        }
    }
    if (!a.part) return;
    float *part = a.part + (size_t)blockIdx.x * 2 * cols;
    if (RPG == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            ln_store<float, V, EDGE>(part, at[c], cols, dw[c]);
            ln_store<float, V, EDGE>(part + cols, at[c], cols, db[c]);
        }
    } else {
        // the rows that the workgroup's teams took side by side are added up in LDS, team 0 first (elements that two
        // threads of a team have are the same in both)
        __shared__ float acc[RPG > 1 ? RPG * TPR * C * V : 1];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            lrb_barrier();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (at[c].any(V)) acc[(threadIdx.x / TPR) * (TPR * C * V) + at[c].at + i] = which ? db[c][i] : dw[c][i];
            lrb_barrier();
            for (int col = threadIdx.x; col < cols; col += THREADS) {
                float s = 0.0f;
#pragma unroll
                for (int r = 0; r < RPG; ++r) s += acc[r * (TPR * C * V) + col];
                part[(size_t)which * cols + col] = s;
            }
        }
    }
}

// Rows too long for the registers of a workgroup: the row is read again for each of its passes, element by element, mostly from beyond
// the L2 (two workgroups a CU of an XCD, with x and dy of 16,384 float32, are 8 MB against its 4).  Measured (float32): forward
// 1678 x 20,001 102 us, backward 2048 x 16,384 109 us and 49 us for dw and db: twice what the bytes take.
template <typename T, bool ACT> __device__ __forceinline__ float ln_at(const ln_args &a, const T *x, long long row, int col, float &f)
{
    const float v = (float)x[col];
    if (!ACT) return v;
    const float k = a.keep ? (a.keep[row * a.cols + col] ? a.keep_scale : 0.0f) : a.keep_scale;
    f = v > 0.0f ? k : a.slope * k; // du/dx
    return ln_act(v, a.slope, k);
}

__device__ __forceinline__ float ln_w_at(const void *w, int w_f32, int col, float dflt, const float *) { return w ? ((const float *)w)[col] : dflt; }
template <typename T> __device__ __forceinline__ float ln_w_at(const void *w, int w_f32, int col, float dflt, const T *)
{
    return !w ? dflt : w_f32 ? ((const float *)w)[col] : (float)((const T *)w)[col];
}

template <typename T, bool ACT> __global__ __launch_bounds__(1024) void ln_fwd_long_kernel(ln_args a)
{
    __shared__ float red[64];
    int flip = 0;
    const float inv = 1.0f / (float)a.cols;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        float s = 0.0f, f;
        for (int c = threadIdx.x; c < a.cols; c += 1024) s = fmaf(ln_at<T, ACT>(a, x, row, c, f), inv, s);
        float mean = ln_sum<1024>(s, red, flip), s2 = 0.0f;
        s = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float e = ln_at<T, ACT>(a, x, row, c, f) - mean;
            s = fmaf(e, inv, s);
            s2 += e * e;
        }
        ln_sum2<1024>(s, s2, red, flip);
        const float rstd = ln_statistics(s, s2 * inv, a.eps, mean);
        if (a.mean && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        T *y = (T *)a.y + row * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += 1024)
            y[c] = (T)((ln_at<T, ACT>(a, x, row, c, f) - mean) * rstd * ln_w_at(a.w, a.w_f32, c, 1.0f, (const T *)nullptr) +
                       ln_w_at(a.b, a.w_f32, c, 0.0f, (const T *)nullptr));
    }
}

template <typename T, bool ACT> __global__ __launch_bounds__(1024) void ln_bwd_long_kernel(ln_args a)
{
    __shared__ float red[64];
    int flip = 0;
    const float inv = 1.0f / (float)a.cols;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride, *dy = (const T *)a.dy + row * a.dy_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f, f = 1.0f;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float g = (float)dy[c] * ln_w_at(a.w, a.w_f32, c, 1.0f, (const T *)nullptr);
            s1 += g;
            s2 += g * ((ln_at<T, ACT>(a, x, row, c, f) - mean) * rstd);
        }
        ln_sum2<1024>(s1, s2, red, flip);
        s1 *= inv, s2 *= inv;
        T *dx = (T *)a.dx + row * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float g = (float)dy[c] * ln_w_at(a.w, a.w_f32, c, 1.0f, (const T *)nullptr);
            const float hat = (ln_at<T, ACT>(a, x, row, c, f) - mean) * rstd;
            float o = (g - s1 - hat * s2) * rstd;
            if (ACT) o = f == 0.0f ? 0.0f : o * f;
            dx[c] = (T)o;
        }
    }
}

// dw, db partial rows of long rows: a thread a column, blockIdx.y a slice of the rows
template <typename T, bool ACT> __global__ __launch_bounds__(256) void ln_cols_long_kernel(ln_args a)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.0f, db = 0.0f, f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = (float)((const T *)a.dy)[row * a.dy_stride + c];
        dw += d * ((ln_at<T, ACT>(a, (const T *)a.x + row * a.x_stride, row, c, f) - a.mean[row]) * a.rstd[row]);
        db += d;
    }
    a.part[(size_t)blockIdx.y * 2 * a.cols + c] = dw;
    a.part[(size_t)blockIdx.y * 2 * a.cols + a.cols + c] = db;
}

// dw[col], db[col] = the partial rows' sums: 32 columns a workgroup, 32 slices of the partial rows side by side
template <typename W> __global__ __launch_bounds__(1024) void ln_join_kernel(const float *__restrict__ part, int groups, int cols, W *__restrict__ dw, W *__restrict__ db)
{
    __shared__ float acc[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, col = blockIdx.x * 32 + x;
    W *out = blockIdx.y ? db : dw;
    if (!out) return;
    float s = 0.0f;
    if (col < cols)
        for (int g = y; g < groups; g += 32) s += part[((size_t)g * 2 + blockIdx.y) * cols + col];
    acc[y][x] = s;
    lrb_barrier();
    if (y == 0 && col < cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += acc[i][x];
        out[col] = (W)s;
    }
}

// How a row is laid over threads: 16, 64, 256 or 1024 of them by its length, at most 16 elements each (registers: a backward
// pass holds five float32 for each, and 1024 threads have 128 registers each).  Rows longer than 16,384, or than 8,192 in a
// backward pass of float32 or with an activation (it would spill): the _long_ kernels.
static int ln_threads(long long cols, int V)
{
    return cols <= 16 * 2 * V ? 16 : cols <= 64 * 16 ? 64 : cols <= 256 * 16 ? 256 : 1024;
}

static bool ln_is_long(long long cols, bool bwd, bool act, int V) { return cols > 1024 * (bwd && (act || V == 4) ? 8 : 16); }

// Workgroups of a pass.  A backward pass writes a partial row of dw and db for each (8 bytes a column), so of long rows it takes
// no more than fill the CUs, and gives each as many rows as the others (1000 rows of 10,007: 250 workgroups of four rows
// write 20 MB of partial rows beside 60 MB of tensors; 1000 of one row would write 80).
static int ln_groups(long long rows, long long cols, int V, bool bwd, bool act)
{
    if (ln_is_long(cols, bwd, act, V)) return (int)(rows < 64 ? (rows ? rows : 1) : 64);
    const int tpr = ln_threads(cols, V), rpg = tpr < 256 ? 256 / tpr : 1;
    const long long turns = (rows + rpg - 1) / rpg, most = bwd && tpr == 1024 ? 256 : LN_MAX_GROUPS;
    if (turns <= most) return (int)(turns ? turns : 1);
    const long long each = (turns + most - 1) / most;
    return (int)((turns + each - 1) / each);
}

template <typename T, bool ACT> static void ln_launch_fwd(const ln_args &a, hipStream_t st)
{
    constexpr int V = ln_vec<T>::V;
    if (ln_is_long(a.cols, false, ACT, V)) {
        hipLaunchKernelGGL((ln_fwd_long_kernel<T, ACT>), dim3((unsigned)(a.rows < 2048 ? a.rows : 2048)), dim3(1024), 0, st, a);
        return;
    }
    const int tpr = ln_threads(a.cols, V), c = (a.cols + tpr * V - 1) / (tpr * V);
    const dim3 grid(ln_groups(a.rows, a.cols, V, false, ACT));
#define LN_GO(TPR, C)                                                                                                       \
    do {                                                                                                                    \
        if (a.cols % V) hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, C, ACT, LN_ODD>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, a); \
        else hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, C, ACT, LN_EVEN>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, a);      \
    } while (0)
#define LN_PICK(TPR, LOW)                \
    if (c <= (LOW)) LN_GO(TPR, (LOW));   \
    else if (c <= 2) LN_GO(TPR, 2);      \
    else LN_GO(TPR, (V == 4 ? 4 : 2))
    if (a.cols < V) {
        hipLaunchKernelGGL((ln_fwd_kernel<T, 16, 1, ACT, LN_TINY>), grid, dim3(256), 0, st, a);
    } else if (tpr == 16) {
        if (c == 1) LN_GO(16, 1);
        else LN_GO(16, 2);
    } else if (tpr == 64) {
        LN_PICK(64, 1);
    } else if (tpr == 256) {
        LN_PICK(256, (V == 4 ? 2 : 1));
    } else {
        LN_PICK(1024, (V == 4 ? 2 : 1));
    }
#undef LN_PICK
#undef LN_GO
}

template <typename T, bool ACT> static void ln_launch_bwd(const ln_args &a, hipStream_t st)
{
    constexpr int V = ln_vec<T>::V;
    if (ln_is_long(a.cols, true, ACT, V)) {
        if (a.dx && a.rows) hipLaunchKernelGGL((ln_bwd_long_kernel<T, ACT>), dim3((unsigned)(a.rows < 2048 ? a.rows : 2048)), dim3(1024), 0, st, a);
        if (a.part)
            hipLaunchKernelGGL((ln_cols_long_kernel<T, ACT>), dim3((a.cols + 255) / 256, ln_groups(a.rows, a.cols, V, true, ACT)), dim3(256), 0, st, a);
        return;
    }
    const int tpr = ln_threads(a.cols, V), c = (a.cols + tpr * V - 1) / (tpr * V);
    const dim3 grid(ln_groups(a.rows, a.cols, V, true, ACT));
#define LN_GO(TPR, C)                                                                                                       \
    do {                                                                                                                    \
        if (a.cols % V) hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, C, ACT, LN_ODD>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, a); \
        else hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, C, ACT, LN_EVEN>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, a);      \
    } while (0)
#define LN_PICK(TPR, LOW)                \
    if (c <= (LOW)) LN_GO(TPR, (LOW));   \
    else if (c <= 2) LN_GO(TPR, 2);      \
    else LN_GO(TPR, (V == 4 ? 4 : 2))
    if (a.cols < V) {
        hipLaunchKernelGGL((ln_bwd_kernel<T, 16, 1, ACT, LN_TINY>), grid, dim3(256), 0, st, a);
    } else if (tpr == 16) {
        if (c == 1) LN_GO(16, 1);
        else LN_GO(16, 2);
    } else if (tpr == 64) {
        LN_PICK(64, 1);
    } else if (tpr == 256) {
        LN_PICK(256, (V == 4 ? 2 : 1));
    } else {
        if (c <= 1 || V == 4) LN_GO(1024, (V == 4 ? 2 : 1));
        else LN_GO(1024, (ACT ? 1 : 2));
    }
#undef LN_PICK
#undef LN_GO
}

extern "C" int lrb_layer_norm_fwd_dev(int device, void *stream, int x_type, int w_type, uint64_t rows, uint64_t cols, const void *d_x,
                                      int64_t x_stride, const void *d_w, const void *d_b, float eps, float slope, const uint8_t *d_keep,
                                      float keep_scale, void *d_y, float *d_mean, float *d_rstd)
{
    ARG_TRY(x_type >= LRB_F32 && x_type <= LRB_F16 && (w_type == LRB_F32 || w_type == x_type));
    ARG_TRY(cols >= 1 && cols <= INT_MAX / 4 && rows <= (1ull << 40));
    ARG_TRY((d_mean == nullptr) == (d_rstd == nullptr));
    if (rows == 0) return LRB_OK;
    ARG_TRY(d_x != nullptr && d_y != nullptr);
    lrb_on_device on(device);
    HIP_TRY(on.err);
    ln_args a = {};
    a.x = d_x, a.w = d_w, a.b = d_b, a.keep = d_keep, a.y = d_y, a.mean = d_mean, a.rstd = d_rstd;
    a.x_stride = x_stride, a.rows = (long long)rows, a.cols = (int)cols, a.w_f32 = w_type == LRB_F32;
    a.eps = eps, a.slope = slope, a.keep_scale = d_keep ? keep_scale : 1.0f;
    const bool act = d_keep || slope != 1.0f;
    hipStream_t st = (hipStream_t)stream;
    if (x_type == LRB_F32) act ? ln_launch_fwd<float, true>(a, st) : ln_launch_fwd<float, false>(a, st);
    else if (x_type == LRB_BF16) act ? ln_launch_fwd<__bf16, true>(a, st) : ln_launch_fwd<__bf16, false>(a, st);
    else act ? ln_launch_fwd<_Float16, true>(a, st) : ln_launch_fwd<_Float16, false>(a, st);
    HIP_TRY(hipGetLastError());
    return LRB_OK;
}

extern "C" uint64_t lrb_layer_norm_bwd_ws_bytes(int x_type, uint64_t rows, uint64_t cols)
{
    if (x_type < LRB_F32 || x_type > LRB_F16 || cols > INT_MAX / 4 || rows > (1ull << 40)) return 0;
    return (uint64_t)ln_groups((long long)rows, (long long)cols, x_type == LRB_F32 ? 4 : 8, true, false) * 2 * cols * sizeof(float);
}

extern "C" int lrb_layer_norm_bwd_dev(int device, void *stream, int x_type, int w_type, uint64_t rows, uint64_t cols, const void *d_x,
                                      int64_t x_stride, const void *d_dy, int64_t dy_stride, const void *d_w, const float *d_mean,
                                      const float *d_rstd, float slope, const uint8_t *d_keep, float keep_scale, void *d_dx, void *d_dw,
                                      void *d_db, void *d_ws, uint64_t ws_bytes)
{
    ARG_TRY(x_type >= LRB_F32 && x_type <= LRB_F16 && (w_type == LRB_F32 || w_type == x_type));
    ARG_TRY(cols >= 1 && cols <= INT_MAX / 4 && rows <= (1ull << 40));
    const bool sums = d_dw || d_db;
    ARG_TRY(!sums || (d_ws != nullptr && ws_bytes >= lrb_layer_norm_bwd_ws_bytes(x_type, rows, cols)));
    ARG_TRY(rows == 0 || (d_x != nullptr && d_dy != nullptr && d_mean != nullptr && d_rstd != nullptr));
    if (!sums && (!d_dx || rows == 0)) return LRB_OK;
    lrb_on_device on(device);
    HIP_TRY(on.err);
    ln_args a = {};
    a.x = d_x, a.dy = d_dy, a.w = d_w, a.keep = d_keep, a.dx = d_dx, a.mean = (float *)d_mean, a.rstd = (float *)d_rstd;
    a.part = sums ? (float *)d_ws : nullptr;
    a.x_stride = x_stride, a.dy_stride = dy_stride, a.rows = (long long)rows, a.cols = (int)cols, a.w_f32 = w_type == LRB_F32;
    a.slope = slope, a.keep_scale = d_keep ? keep_scale : 1.0f;
    const bool act = d_keep || slope != 1.0f;
    hipStream_t st = (hipStream_t)stream;
    if (x_type == LRB_F32) act ? ln_launch_bwd<float, true>(a, st) : ln_launch_bwd<float, false>(a, st);
    else if (x_type == LRB_BF16) act ? ln_launch_bwd<__bf16, true>(a, st) : ln_launch_bwd<__bf16, false>(a, st);
    else act ? ln_launch_bwd<_Float16, true>(a, st) : ln_launch_bwd<_Float16, false>(a, st);
    if (sums) {
        const int groups = ln_groups(a.rows, a.cols, x_type == LRB_F32 ? 4 : 8, true, act);
        const dim3 grid((a.cols + 31) / 32, 2);
        if (w_type == LRB_F32) hipLaunchKernelGGL((ln_join_kernel<float>), grid, dim3(1024), 0, st, (const float *)d_ws, groups, a.cols, (float *)d_dw, (float *)d_db);
        else if (w_type == LRB_BF16) hipLaunchKernelGGL((ln_join_kernel<__bf16>), grid, dim3(1024), 0, st, (const float *)d_ws, groups, a.cols, (__bf16 *)d_dw, (__bf16 *)d_db);
        else hipLaunchKernelGGL((ln_join_kernel<_Float16>), grid, dim3(1024), 0, st, (const float *)d_ws, groups, a.cols, (_Float16 *)d_dw, (_Float16 *)d_db);
    }
    HIP_TRY(hipGetLastError());
    return LRB_OK;
}
