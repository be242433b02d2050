// Group normalisation with an activation over channels-last tensors x [B, S, C], S positions, C = G D channels in G groups:
//     mean, var over the S D elements of a sample's group;   xhat = (x - mean) / sqrt(var + eps)
//     z = xhat gamma[c] + beta[c];   y = act(z)
// Backward, with dz = dy act'(z) and d = dz gamma:
//     dx = (d - mean(d) - xhat mean(d xhat)) / sqrt(var + eps);   dgamma[c] = sum dz xhat,  dbeta[c] = sum dz  over B and S
// x, y, dy and dx have one of three types; everything between is fp32, the variance about the mean (not a difference of squares).
//
// The border of a relu.  Which side of zero z falls on decides whether a whole dy passes, and z within fp32's rounding of zero (one element in
// some ten million) decides it by chance, for every evaluation in fp32 its own.  So before a relu mean and 1 / sqrt(var + eps) are formed in 64 bits
// and handed to the backward pass as such, and what the mean's rounding to fp32 left out goes into the forward pass's beta (far from zero it would move
// the border: at a mean of 3000 standard deviations by 1e-4 of one); backward z > 0 is x > t (x < t where gamma is negative) with t = mean - beta / (gamma rstd),
// rounded to fp32 towards the side that changes no comparison with an fp32 x: the exact decision takes fewer instructions than z.
#include <type_traits>

#include "hgq_device.h"
#include "hgq_host.h"

namespace hgq {

struct GroupShape {
    int64_t B, S;
    int C, G, D;
    float eps;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<_Float16>(_Float16 v) {
    return (float)v;
}
template <>
__device__ __forceinline__ float to_f32<__bf16>(__bf16 v) {
    return (float)v;
}

// 1 / (1 + exp(-z)).  The product z / ln 2 is off by half a unit, so exp(-z) relatively by |z| 2^-24; 1 / inf = 0 where it overflows.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269502f)); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == HGQ_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if (ACT == HGQ_ACT_SILU) return z * sigmoid(z);
    return z;
}

// Before a relu: z > 0 where x - t has the sign of scale = gamma rstd; a difference of zero counts as positive, so t is the smallest number that passes
// for a positive scale, and the last one that does not below a negative one, -0 where it is zero (x - t is then +0 for both zeros).  Signs, not
// their product: that may underflow.  A gamma of zero leaves beta alone to decide, by the sign of an infinite t; what is not a number does not pass.
struct ReluBorder {
    float t, scale;
    __device__ __forceinline__ void set(double mean, double rstd, float gamma, float beta) {
        const double a = rstd * gamma;
        scale = (float)a;
        if (scale == 0.0f) scale = a < 0.0 ? -0x1p-149f : 0x1p-149f;  // (of the sign that fp32 would lose)
        double inv = __builtin_amdgcn_rcp(a);  // and two steps of Newton's: a rounded division and rounding by library calls took 1 us a wavefront
        inv = fma(fma(-a, inv, 1.0), inv, inv), inv = fma(fma(-a, inv, 1.0), inv, inv);
        const double at = fma(-(double)beta, inv, mean);
        t = (float)at;
        if (a > 0.0 ? (double)t <= at : (double)t < at) {  // the next one up
            const int bits = __float_as_int(t);
            if (t < INFINITY) t = t == 0.0f ? 0x1p-149f : __int_as_float(t > 0.0f ? bits + 1 : bits - 1);
        }
        if (a == 0.0) t = beta > 0.0f ? -INFINITY : INFINITY;
        if (!(t == t && a == a)) t = a < 0.0 ? -INFINITY : INFINITY, scale = fabsf(scale) >= 0.0f ? scale : __builtin_nanf("");
        if (t == 0.0f) t = -0.0f;
    }
    __device__ __forceinline__ float through(float dy, float x) const { return (__float_as_int(x - t) ^ __float_as_int(scale)) >= 0 ? dy : 0.0f; }
};

// dy act'(z), of silu and of no activation
template <int ACT>
__device__ __forceinline__ float through_activation(float dy, float z) {
    if (ACT == HGQ_ACT_SILU) {
        const float p = sigmoid(z);
        return dy * (p * fmaf(z, 1.0f - p, 1.0f));
    }
    return dy;
}

// sum of the workgroup's values in a fixed order, to every thread
__device__ __forceinline__ double group_sum(double v, double *lds) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) v += lds[w];
    __syncthreads();
    return v;
}

// A workgroup takes one sample's group after another, any shape: the group is read three times, its sums are formed in fp64.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void group_norm_fwd_any(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                                          T *__restrict__ y, double *__restrict__ mean_out, double *__restrict__ rstd_out, GroupShape s) {
    __shared__ double lds[4];
    for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
        const int64_t b = bg / s.G;
        const int g = (int)(bg - b * s.G);
        const int64_t base = b * s.S * s.C + (int64_t)g * s.D, n = s.S * s.D;
        double sum = 0;
        for (int64_t e = threadIdx.x; e < n; e += 256) sum += to_f32(x[base + e / s.D * s.C + e % s.D]);
        const double mean64 = group_sum(sum, lds) / (double)n;
        const float mean = (float)mean64;
        double sq = 0;
        for (int64_t e = threadIdx.x; e < n; e += 256) {
            const double d = to_f32(x[base + e / s.D * s.C + e % s.D]) - mean64;
            sq += d * d;
        }
        const double rstd64 = 1.0 / sqrt(group_sum(sq, lds) / (double)n + s.eps);
        const float rstd = (float)rstd64;
        if (threadIdx.x == 0) mean_out[bg] = mean64, rstd_out[bg] = rstd64;
        for (int64_t e = threadIdx.x; e < n; e += 256) {
            const int c = g * s.D + (int)(e % s.D);
            const int64_t at = base + e / s.D * s.C + e % s.D;
            const float scale = rstd * (gamma ? gamma[c] : 1.0f);
            float be = beta ? beta[c] : 0.0f;
            if (ACT == HGQ_ACT_RELU) be = fmaf(-(float)(mean64 - mean), scale, be);
            y[at] = (T)activate<ACT>(fmaf(to_f32(x[at]) - mean, scale, be));
        }
    }
}

// A workgroup takes one sample's group after another, any shape.  part [B][2 C]: each sample's terms of dgamma, then of dbeta.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void group_norm_bwd_any(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                          const float *__restrict__ beta, const double *__restrict__ mean_in,
                                                          const double *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ part, GroupShape s) {
    __shared__ double lds[4];
    __shared__ double col[2][256];
    int tx = 1;  // threads side by side over channels, the others over positions
    while (tx < s.D && tx < 256) tx *= 2;
    const int ty = 256 / tx, cx = threadIdx.x % tx, py = threadIdx.x / tx;
    for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
        const int64_t b = bg / s.G;
        const int g = (int)(bg - b * s.G);
        const int64_t base = b * s.S * s.C + (int64_t)g * s.D, n = s.S * s.D;
        const float mean = (float)mean_in[bg], rstd = (float)rstd_in[bg];
        auto border = [&](float ga, float be) {
            ReluBorder r = {0, 0};
            if (ACT == HGQ_ACT_RELU) r.set(mean_in[bg], rstd_in[bg], ga, be);
            return r;
        };
        auto through = [&](float dv, float xv, float xh, float ga, float be, const ReluBorder &edge) {  // dz
            if (ACT != HGQ_ACT_RELU) return through_activation<ACT>(dv, xh * ga + be);
            return xh == xh ? edge.through(dv, xv) : xh;
        };
        double s1 = 0, s2 = 0;  // of d and d xhat, over the group
        for (int c0 = 0; c0 < s.D; c0 += tx) {
            const int d = c0 + cx, c = g * s.D + d;
            double a = 0, h = 0;
            const float ga = d < s.D && gamma ? gamma[c] : 1.0f, be = d < s.D && beta ? beta[c] : 0.0f;
            const ReluBorder edge = border(ga, be);
            if (d < s.D)
                for (int64_t p = py; p < s.S; p += ty) {
                    const int64_t at = base + p * s.C + d;
                    const float xv = to_f32(x[at]), xh = (xv - mean) * rstd;
                    const float dz = through(to_f32(dy[at]), xv, xh, ga, be, edge);
                    a += dz, h += (double)dz * xh;
                }
            s1 += a * ga, s2 += h * ga;
            col[0][threadIdx.x] = h, col[1][threadIdx.x] = a;
            __syncthreads();
            if (py == 0 && d < s.D && part) {
                for (int r = 1; r < ty; ++r) h += col[0][r * tx + cx], a += col[1][r * tx + cx];
                part[b * 2 * s.C + c] = (float)h, part[b * 2 * s.C + s.C + c] = (float)a;
            }
            __syncthreads();
        }
        const float m1 = (float)(group_sum(s1, lds) / (double)n), m2 = (float)(group_sum(s2, lds) / (double)n);
        if (!dx) continue;
        for (int64_t e = threadIdx.x; e < n; e += 256) {
            const int c = g * s.D + (int)(e % s.D);
            const int64_t at = base + e / s.D * s.C + e % s.D;
            const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f, xv = to_f32(x[at]), xh = (xv - mean) * rstd;
            const float dz = through(to_f32(dy[at]), xv, xh, ga, be, border(ga, be));
            dx[at] = (T)((dz * ga - m1 - xh * m2) * rstd);
        }
    }
}


// ---- tiles held in registers -----------------------------------------------------------------------------------------
// A workgroup holds a tile - the positions (or a run of them) of K whole groups of one sample, or of several small samples - in
// registers, four neighbours per access, so x (and dy) are read once and the variance is formed about the mean in a second
// pass over registers.  A thread keeps its four columns in all its rows, and with them its scales and its sums per channel.
// Rows: positions (K < G: rows of C channels of which K D are the tile's); with all groups, q = 4 / gcd(C, 4) positions are one
// row, so rows are whole accesses for every C; the last row may be short.  A sample that is too long for one tile is cut into
// `splits` runs of rows: one launch leaves their sums, the next one joins them and applies them.
struct GroupTile {
    int64_t B;
    int n, C, G, D, K, stride;       // n: elements of a sample; stride: of a row
    int fold;                        // positions per row
    int TX, TY, NS;                  // threads across a row; rows of a sample side by side; samples
    int rows, split_rows, splits;    // rows of a sample; of a split
    int chunks, tiles;               // G / K; runs of rows (or sets of samples) of all samples
    int team;                        // threads that add up a group's sums
    bool through;                    // the output is more than the cache keeps: it is written past it
    float eps, inv;                  // 1 / elements of a group
};

// four neighbours as they lie in memory: sizeof(T) words
template <typename T>
struct Four {
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(T))));
    typedef words unaligned __attribute__((aligned(sizeof(T))));
    words w;

    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(&w, p, sizeof(w)); }  // (rows of any width: aligned to an element only)
    __device__ __forceinline__ void load_last(const T *p) {  // past the cache
        w = __builtin_nontemporal_load((const unaligned *)p);
    }
    __device__ __forceinline__ void store(T *p, bool through) const {  // through: past the cache
        if (through) __builtin_nontemporal_store(w, (unaligned *)p);
        else __builtin_memcpy(p, &w, sizeof(w));
    }
    __device__ __forceinline__ float get(int j) const {
        T v[4];
        __builtin_memcpy(v, &w, sizeof(w));
        return to_f32(v[j]);
    }
    __device__ __forceinline__ void set(const float (&f)[4]) {
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (T)f[j];
        __builtin_memcpy(&w, v, sizeof(w));
    }
    // What is cheap to form again is not carried in registers from one pass over the tile to the next: the compiler forgets what it knows.
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w)); }
};

// where a thread works: its sample in the tile, row and columns
struct GroupThread {
    int s, ty, col;
    bool on;
    __device__ __forceinline__ explicit GroupThread(const GroupTile &p) {
        const int tx = threadIdx.x % p.TX, rr = threadIdx.x / p.TX;
        s = rr / p.TY, ty = rr - s * p.TY, col = tx * 4, on = s < p.NS;
    }
};

// A thread's accesses of a run of rows [r0, r1): `full` whole ones from element `at` of the sample on, `step` apart, then `rest` elements
struct GroupRows {
    int full, rest, at, step;
    __device__ __forceinline__ GroupRows(const GroupTile &p, const GroupThread &t, bool on, int c0, int r0, int r1) {
        const int r = r0 + t.ty, rows = on && r < r1 ? (r1 - r + p.TY - 1) / p.TY : 0;
        at = r * p.stride + c0, step = p.TY * p.stride, full = rows, rest = 0;
        if (rows > 0) {
            const int behind = at + (rows - 1) * step + 4 - p.n;  // (only a sample's last row is short)
            if (behind > 0) full = rows - 1, rest = behind < 4 ? 4 - behind : 0;
        }
    }
};

// Sums of one value per column (v[4] of each thread) over the rows and the columns of every group in the tile: total[NS * K] in LDS, to
// all threads, in a fixed order.  ONE: a thread's columns are of one group, and it adds them first.  red: blockDim.x * (ONE ? 1 : 4).
template <bool ONE, typename V>
__device__ __forceinline__ void sum_groups(const GroupTile &p, const GroupThread &t, const V (&v)[4], V *red, V *total) {
    if (t.on) {
        if (ONE) {
            red[threadIdx.x] = (v[0] + v[1]) + (v[2] + v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) red[threadIdx.x * 4 + j] = v[j];
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & (p.team - 1);
    const int across = ONE ? p.D / 4 : p.D, width = ONE ? p.TX : p.TX * 4, cols = ONE ? across : across * p.fold;
    const int r0 = lane / cols, first = lane - r0 * cols, step = p.team / cols, rest = p.team - step * cols;
    for (int g = threadIdx.x / p.team; g < p.NS * p.K; g += blockDim.x / p.team) {
        const V *mine = red + (g / p.K) * p.TY * width + (g % p.K) * across;
        V sum = 0;
        for (int r = r0, c = first; r < p.TY;) {
            const int f = !ONE && p.fold > 1 ? c / across : 0;
            sum += mine[r * width + f * p.C + (c - f * across)];
            r += step, c += rest;
            if (c >= cols) c -= cols, ++r;
        }
        for (int d = p.team / 2; d; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) total[g] = sum;
    }
    __syncthreads();
}

// the group of a thread's column j within the tile
template <bool ONE>
__device__ __forceinline__ int group_of(const GroupTile &p, const GroupThread &t, int j) {
    const int c = t.col + (ONE ? 0 : j);
    return t.s * p.K + (!ONE && p.fold > 1 ? c % p.C : c) / p.D;
}

// phase 0: whole tiles; 1: mean and sum of squares about it of every split, parts [B][splits][G][2]; 2: join those, apply
template <typename T, int ACT, bool ONE, int NV>
__global__ __launch_bounds__(1024) void group_norm_fwd_tile(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                                            T *__restrict__ y, double *__restrict__ mean_out, double *__restrict__ rstd_out,
                                                            double *__restrict__ parts, GroupTile p, int phase) {
    typedef std::conditional_t<ACT == HGQ_ACT_RELU, double, float> V;  // of the sums and what they give
    extern __shared__ float lds[];
    const int groups = p.NS * p.K;
    V *total = (V *)lds, *stat = total + groups, *red = stat + groups;
    const GroupThread t(p);
    // the chunks of one sample share cache lines: their workgroups follow each other on one of the eight dies (blocks go round them)
    const int64_t blk = blockIdx.x;
    const int64_t z = blk / (8 * p.chunks) * 8 + blk % 8;
    const int chunk = (int)(blk / 8 % p.chunks);
    if (z >= p.tiles) return;
    const int split = (int)(z % p.splits);
    const int64_t b = z / p.splits * p.NS + t.s;
    const bool on = t.on && b < p.B;
    const int c0 = chunk * p.K * p.D + t.col;  // (with fold: the column in the row)
    const int r0 = split * p.split_rows, r1 = min(p.rows, r0 + p.split_rows);
    const T *xs = x + b * p.n;
    const GroupRows rows(p, t, on, c0, r0, r1);
    Four<T> v[NV];
    float last[3] = {0, 0, 0};
    if (phase == 2 && p.through) {  // (the last read of what the cache does not keep)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) v[i].load_last(xs + rows.at + i * rows.step);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) v[i].load(xs + rows.at + i * rows.step);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < rows.rest) last[j] = to_f32(xs[rows.at + rows.full * rows.step + j]);
    constexpr int N = ONE ? 1 : 4;  // means of a thread's columns
    float mean[N], rstd[N];
    const V one = 1, eps = p.eps;
    // elements of a group in this tile
    const V inv = one / (V)(p.splits == 1 ? p.n / p.G : (min(p.n / p.C, r1 * p.fold) - r0 * p.fold) * p.D);
    if (phase < 2) {
        V acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += v[i].get(j);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) acc[j] += last[j];
        sum_groups<ONE>(p, t, acc, red, total);
#pragma unroll
        for (int j = 0; j < N; ++j) mean[j] = t.on ? (float)(total[group_of<ONE>(p, t, j)] * inv) : 0.0f;
        auto square = [&](float x, int j) {  // (about the mean's fp32 value: within 2^-24 of it, whose square is nothing)
            const V d = x - mean[j % N];
            acc[j] = fma(d, d, acc[j]);
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) {
                v[i].forget();
#pragma unroll
                for (int j = 0; j < 4; ++j) square(v[i].get(j), j);
            }
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) square(last[j], j);
        sum_groups<ONE>(p, t, acc, red, stat);
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            const int64_t bg = z / p.splits * p.NS + g / p.K;
            if (bg >= p.B) break;
            const int64_t at = bg * p.G + chunk * p.K + g % p.K;
            if (phase == 1) {
                double *out = parts + ((bg * p.splits + split) * p.G + chunk * p.K + g % p.K) * 2;
                out[0] = total[g] * inv, out[1] = stat[g];
            } else {
                mean_out[at] = total[g] * inv, rstd_out[at] = one / sqrt(stat[g] * inv + eps);
            }
        }
        if (phase == 1) return;
#pragma unroll
        for (int j = 0; j < N; ++j) rstd[j] = t.on ? (float)(one / sqrt(stat[group_of<ONE>(p, t, j)] * inv + eps)) : 0.0f;
    } else {
        // the splits' means, and their squares about the joint one
        const int lane = threadIdx.x & (p.team - 1);
        for (int g = threadIdx.x / p.team; g < groups; g += blockDim.x / p.team) {
            const double *in = parts + (b - t.s) * p.splits * p.G * 2 + (chunk * p.K + g) * 2;  // (one sample: NS = 1)
            const double all = 1.0 / (double)(p.n / p.G);
            auto share = [&](int k) { return (double)((min(p.n / p.C, (k + 1) * p.split_rows * p.fold) - k * p.split_rows * p.fold) * p.D) * all; };
            double m = 0, q = 0;
            for (int k = lane; k < p.splits; k += p.team) m += share(k) * in[(int64_t)k * p.G * 2];
            for (int d = p.team / 2; d; d >>= 1) m += __shfl_xor(m, d);
            for (int k = lane; k < p.splits; k += p.team) {
                const double d = in[(int64_t)k * p.G * 2] - m;
                q += in[(int64_t)k * p.G * 2 + 1] * all + share(k) * d * d;
            }
            for (int d = p.team / 2; d; d >>= 1) q += __shfl_xor(q, d);
            if (lane == 0) {
                const double r = 1.0 / sqrt(q + (double)p.eps);
                total[g] = (V)m, stat[g] = (V)r;
                if (split == 0) mean_out[(b - t.s) * p.G + chunk * p.K + g] = m, rstd_out[(b - t.s) * p.G + chunk * p.K + g] = r;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) mean[j] = t.on ? (float)total[group_of<ONE>(p, t, j)] : 0.0f, rstd[j] = t.on ? (float)stat[group_of<ONE>(p, t, j)] : 0.0f;
    }
    if (!on) return;
    float scale[4], be[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = p.fold > 1 ? (c0 + j) % p.C : c0 + j;
        scale[j] = rstd[j % N] * (gamma ? gamma[c] : 1.0f), be[j] = beta ? beta[c] : 0.0f;
        if (ACT == HGQ_ACT_RELU) {  // (the 64-bit mean again from LDS: kept, it took up to eight registers)
            const V m = total[group_of<ONE>(p, t, j)];
            be[j] = fmaf(-(float)((phase < 2 ? m * inv : m) - mean[j % N]), scale[j], be[j]);
        }
    }
    T *ys = y + b * p.n;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i < rows.full) {
            v[i].forget();
            float out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = activate<ACT>(fmaf(v[i].get(j) - mean[j % N], scale[j], be[j]));
            v[i].set(out);
            v[i].store(ys + rows.at + i * rows.step, p.through);
        }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < rows.rest) ys[rows.at + rows.full * rows.step + j] = (T)activate<ACT>(fmaf(last[j] - mean[j % N], scale[j], be[j]));
}

// phase 0: whole tiles; 1: sums of d rstd and d xhat rstd of every split, parts [B][splits][G][2], and the channels' sums; 2: join them, dx.
// Every tile leaves its terms of dgamma and dbeta, slices [tiles][2 C] (NULL: not wanted).  MORE: rows of a thread beyond those in its registers, which it
// keeps in LDS.  The 16-bit forms with 16 rows before a relu, for groups that are not whole accesses, spill 8 of 128 registers (2048 x 26 x 26 x 30
// bfloat16 in 5 groups, backward 75 us; x 32 in 4 groups, without a spill, 65 us).
template <typename T, int ACT, bool ONE, int NV, int MORE>
__global__ __launch_bounds__(MORE ? 512 : 1024, 4) void group_norm_bwd_tile(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                            const float *__restrict__ beta, const double *__restrict__ mean_in,
                                                            const double *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ slices,
                                                            float *__restrict__ parts, GroupTile p, int phase) {
    extern __shared__ float lds[];
    const int groups = p.NS * p.K;
    float *total = lds, *stat = lds + groups, *red = lds + 2 * groups;
    const GroupThread t(p);
    const int64_t blk = blockIdx.x;
    const int64_t z = blk / (8 * p.chunks) * 8 + blk % 8;
    const int chunk = (int)(blk / 8 % p.chunks);
    if (z >= p.tiles) return;
    const int c0 = chunk * p.K * p.D + t.col;
    const int split = (int)(z % p.splits);
    const int64_t b = z / p.splits * p.NS + t.s;
    const bool on = t.on && b < p.B;
    const int r0 = split * p.split_rows, r1 = min(p.rows, r0 + p.split_rows);
    const T *xs = x + b * p.n, *ds = dy + b * p.n;
    const GroupRows rows(p, t, on, c0, r0, r1);
    // A relu's borders, one per column and sample: shared out over the threads and handed on through LDS (every thread for its own four columns:
    // 1024 x 26 x 26 x 32, 57 us for 53); asked for ahead of the tile.
    const int width = p.TX * 4, borders = ACT == HGQ_ACT_RELU && p.TY > 1 ? p.NS * width : 0;
    struct {
        double mean = 0, rstd = 0;
        float gamma = 1, beta = 0;
    } its;
    auto ask = [&](int k) {
        const int col = k % width, c = p.fold > 1 ? col % p.C : chunk * p.K * p.D + col;
        const int64_t of = z / p.splits * p.NS + k / width;
        if (of >= p.B) return;
        const int64_t g = of * p.G + c / p.D;
        its.mean = mean_in[g], its.rstd = rstd_in[g];
        if (gamma) its.gamma = gamma[c];
        if (beta) its.beta = beta[c];
    };
    if ((int)threadIdx.x < borders) ask(threadIdx.x);
    Four<T> v[NV], w[NV], more_v[MORE ? MORE : 1], more_w[MORE ? MORE : 1];
    auto *const kept = (typename Four<T>::words *)(lds + ((2 * groups + 4 * blockDim.x + 3) & ~3u)) + threadIdx.x;  // [MORE][x, dy][threads]
#pragma unroll
    for (int i = 0; i < MORE; ++i)
        if (NV + i < rows.full) more_v[i].load(xs + rows.at + (NV + i) * rows.step), more_w[i].load(ds + rows.at + (NV + i) * rows.step);
    float last[3] = {0, 0, 0}, dlast[3] = {0, 0, 0};
    if (phase == 2 && p.through) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) v[i].load_last(xs + rows.at + i * rows.step), w[i].load_last(ds + rows.at + i * rows.step);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) v[i].load(xs + rows.at + i * rows.step), w[i].load(ds + rows.at + i * rows.step);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < rows.rest) last[j] = to_f32(xs[rows.at + rows.full * rows.step + j]), dlast[j] = to_f32(ds[rows.at + rows.full * rows.step + j]);
#pragma unroll
    for (int i = 0; i < MORE; ++i)
        if (NV + i < rows.full) kept[2 * i * blockDim.x] = more_v[i].w, kept[(2 * i + 1) * blockDim.x] = more_w[i].w;
    constexpr int N = ONE ? 1 : 4;  // groups of a thread's columns
    float mean[N], rstd[N], scale[4], be[4];
    ReluBorder relu[4];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int64_t g = b * p.G + chunk * p.K + group_of<ONE>(p, t, j) - t.s * p.K;
        mean[j] = on ? (float)mean_in[g] : 0.0f, rstd[j] = on ? (float)rstd_in[g] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = p.fold > 1 ? (c0 + j) % p.C : c0 + j;
        const float ga = t.on && gamma ? gamma[c] : 1.0f;
        be[j] = t.on && beta ? beta[c] : 0.0f, scale[j] = rstd[j % N] * ga;
        relu[j].t = relu[j].scale = 0;
        if (ACT == HGQ_ACT_RELU && on && !borders) {
            const int64_t g = b * p.G + chunk * p.K + group_of<ONE>(p, t, j) - t.s * p.K;
            relu[j].set(mean_in[g], rstd_in[g], ga, be[j]);
        }
    }
    if (borders) {
        for (int k = threadIdx.x; k < borders; k += blockDim.x) {
            if (k != (int)threadIdx.x) ask(k);
            ReluBorder it;
            it.set(its.mean, its.rstd, its.gamma, its.beta);
            red[2 * k] = it.t, red[2 * k + 1] = it.scale;
        }
        __syncthreads();
        if (on)
#pragma unroll
            for (int j = 0; j < 4; ++j) relu[j] = {red[2 * (t.s * width + t.col + j)], red[2 * (t.s * width + t.col + j) + 1]};
        __syncthreads();
    }
    auto times = [&](int j) { return ACT == HGQ_ACT_RELU ? relu[j].scale : scale[j]; };  // rstd gamma
    auto through = [&](float dv, float xv, float d, int j) {  // dz
        if (ACT == HGQ_ACT_RELU) return relu[j].through(dv, xv);
        return through_activation<ACT>(dv, fmaf(d, scale[j], be[j]));
    };
    float h[4] = {0, 0, 0, 0}, a[4] = {0, 0, 0, 0};  // of dz (x - mean) and of dz
    if (phase < 2) {
        float mine[2][4];
        auto add = [&](float xv, float dv, int j) {
            const float d = xv - mean[j % N], dz = through(dv, xv, d, j);
            a[j] += dz, h[j] = fmaf(dz, d, h[j]);
        };
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full)
#pragma unroll
                for (int j = 0; j < 4; ++j) add(v[i].get(j), w[i].get(j), j);
        for (int i = 0; i < MORE && NV + i < rows.full; ++i) {
            const Four<T> x4 = {kept[2 * i * blockDim.x]}, d4 = {kept[(2 * i + 1) * blockDim.x]};
#pragma unroll
            for (int j = 0; j < 4; ++j) add(x4.get(j), d4.get(j), j);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) add(last[j], dlast[j], j);
        if (ACT == HGQ_ACT_RELU)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = fmaf(0.0f, mean[j % N], a[j]);  // (a sample that is not finite)
        // sums of d rstd and of d xhat rstd: gamma rstd is what is at hand
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] *= rstd[j % N], mine[0][j] = a[j] * times(j), mine[1][j] = h[j] * times(j);
        if (phase == 1 || dx) {
            sum_groups<ONE>(p, t, mine[0], red, total);
            sum_groups<ONE>(p, t, mine[1], red, stat);
        }
        if (phase == 1) {
            for (int g = threadIdx.x; g < groups; g += blockDim.x) {  // (one sample: NS = 1)
                float *out = parts + (((b - t.s) * p.splits + split) * p.G + chunk * p.K + g) * 2;
                out[0] = total[g], out[1] = stat[g];
            }
        }
    } else {
        const int lane = threadIdx.x & (p.team - 1);
        for (int g = threadIdx.x / p.team; g < groups; g += blockDim.x / p.team) {
            const float *in = parts + (b - t.s) * p.splits * p.G * 2 + (chunk * p.K + g) * 2;
            double m1 = 0, m2 = 0;  // (thousands of splits in a row: in fp32 they drift by hundreds of its roundings)
            for (int k = lane; k < p.splits; k += p.team) m1 += in[(int64_t)k * p.G * 2], m2 += in[(int64_t)k * p.G * 2 + 1];
            for (int d = p.team / 2; d; d >>= 1) m1 += __shfl_xor(m1, d), m2 += __shfl_xor(m2, d);
            if (lane == 0) total[g] = (float)m1, stat[g] = (float)m2;
        }
        __syncthreads();
    }
    if (phase != 1 && dx && on) {
        // dx = dz gamma rstd - mean(d) rstd - (x - mean) rstd mean(d xhat) rstd
        float m1[N], m2[N];
#pragma unroll
        for (int j = 0; j < N; ++j) m1[j] = -total[group_of<ONE>(p, t, j)] * p.inv, m2[j] = -stat[group_of<ONE>(p, t, j)] * p.inv * rstd[j];
        T *out = dx + b * p.n;
        auto one = [&](float xv, float dv, int j) {
            const float d = xv - mean[j % N];
            return fmaf(through(dv, xv, d, j), times(j), fmaf(d, m2[j % N], m1[j % N]));
        };
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) {
                v[i].forget(), w[i].forget();
                float o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = one(v[i].get(j), w[i].get(j), j);
                v[i].set(o);
                v[i].store(out + rows.at + i * rows.step, p.through);
            }
        for (int i = 0; i < MORE && NV + i < rows.full; ++i) {
            Four<T> x4 = {kept[2 * i * blockDim.x]};
            const Four<T> d4 = {kept[(2 * i + 1) * blockDim.x]};
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = one(x4.get(j), d4.get(j), j);
            x4.set(o);
            x4.store(out + rows.at + (NV + i) * rows.step, p.through);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) out[rows.at + rows.full * rows.step + j] = (T)one(last[j], dlast[j], j);
    }
    if (!slices || phase == 2) return;
    // this tile's sums per channel: over its rows and samples, the folded positions with them
    const int cols = p.K * p.D, folds = p.fold == 4 ? 2 : p.fold - 1, count = (p.NS * p.TY) << folds;  // (fold = 1, 2 or 4)
    int team = 1;
    while (team < 64 && team * 2 * cols <= (int)blockDim.x) team *= 2;
    const int lane = threadIdx.x & (team - 1);
    for (int k = 0; k < 2; ++k) {
        if (t.on)
#pragma unroll
            for (int j = 0; j < 4; ++j) red[threadIdx.x * 4 + j] = k ? a[j] : h[j];
        __syncthreads();
        for (int c = threadIdx.x / team; c < cols; c += blockDim.x / team) {
            float sum = 0;
            for (int e = lane; e < count; e += team) sum += red[(e >> folds) * width + (e & (p.fold - 1)) * p.C + c];
            for (int d = team / 2; d; d >>= 1) sum += __shfl_xor(sum, d);
            if (lane == 0) slices[z * 2 * p.C + k * p.C + chunk * cols + c] = sum;
        }
        __syncthreads();
    }
}

// Adds up runs of SLICE_RUN slices of M entries: where a batch leaves more slices than the last reduction takes well.  All loads of a run are in
// flight at once (20000 x 30 x 48 in 6 groups, 10000 slices: runs of 64 by eight loads 22 us, of 32 by 32 loads 4.3 us).
constexpr int SLICE_RUN = 32;
__global__ __launch_bounds__(64) void group_norm_join_slices(const float *__restrict__ slices, int64_t n, int64_t M, float *__restrict__ out) {
    const int64_t e = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (e >= M) return;
    for (int64_t run = blockIdx.y; run * SLICE_RUN < n; run += gridDim.y) {
        const int64_t first = run * SLICE_RUN, behind = n - first;
        float v[SLICE_RUN];
#pragma unroll
        for (int k = 0; k < SLICE_RUN; ++k) v[k] = k < behind ? slices[(first + k) * M + e] : 0.0f;
#pragma unroll
        for (int d = SLICE_RUN / 2; d; d /= 2)
#pragma unroll
            for (int k = 0; k < d; ++k) v[k] += v[k + d];
        out[run * M + e] = v[0];
    }
}

}  // namespace hgq

using namespace hgq;

namespace {

int check_shape(const char *what, int64_t B, int64_t S, int C, int G, int act, int type) {
    if (B < 0 || S < 0 || C < 1 || G < 1 || C % G) return fail(HGQ_ERR_ARG, "%s: bad shape [%lld, %lld, %d] in %d groups", what, (long long)B, (long long)S, C, G);
    if (S > 0 && B > ((int64_t)1 << 46) / S / C) return fail(HGQ_ERR_ARG, "%s: too many elements", what);
    if (B > 0x7fffffff / G) return fail(HGQ_ERR_UNSUPPORTED, "%s: more than 2^31 groups", what);
    if (act != HGQ_ACT_NONE && act != HGQ_ACT_RELU && act != HGQ_ACT_SILU) return fail(HGQ_ERR_ARG, "%s: unknown activation", what);
    if (type != HGQ_TYPE_F32 && type != HGQ_TYPE_BF16 && type != HGQ_TYPE_F16) return fail(HGQ_ERR_ARG, "%s: unknown type", what);
    return HGQ_OK;
}

constexpr int GROUP_THREADS = 1024;  // most threads of a workgroup
constexpr int64_t MOST_SLICES = 2048;

// accesses of four that a thread can hold of one tensor: 128 bytes
template <typename T>
constexpr int MOST_HELD = 32 / sizeof(T);
int most_held(int type) { return type == HGQ_TYPE_F32 ? MOST_HELD<float> : MOST_HELD<__bf16>; }
// and further ones in LDS (backward, both tensors): 48 KB of a workgroup of 512 threads
constexpr int in_lds(int most) { return 3 * most / 8; }

// The tile's width for K of the groups; false: it is none (more than GROUP_THREADS accesses, or not whole ones)
bool widen(GroupTile &p, int K) {
    if (K > 1024) return false;  // (their sums lie in LDS)
    p.K = K;
    p.fold = K < p.G ? 1 : p.C % 4 == 0 ? 1 : p.C % 2 == 0 ? 2 : 4;
    if (K < p.G && (int64_t)K * p.D % 4) return false;
    const int64_t width = K < p.G ? (int64_t)K * p.D : (int64_t)p.fold * p.C;
    if (width > 4 * GROUP_THREADS) return false;
    p.TX = (int)(width / 4);
    p.stride = K < p.G ? p.C : (int)width;
    const int S = p.n / p.C;
    p.rows = (S + p.fold - 1) / p.fold;
    p.chunks = p.G / K;
    return true;
}

// Lays out the tiles; false: the shape is left to the kernels for any shape.  held: accesses per thread.
bool plan(GroupTile &p, int &held, int &threads, int64_t B, int64_t S, int C, int G, int type, bool backward) {
    if (B == 0 || S == 0 || S > (1 << 29) / C || C > 65536) return false;  // (offsets within a sample, and a tile behind it, in 32 bits)
    p = {};
    p.B = B, p.n = (int)(S * C), p.C = C, p.G = G, p.D = C / G, p.inv = 1.0f / (float)(S * (C / G)), p.NS = 1;
    const int most = most_held(type), size = type == HGQ_TYPE_F32 ? 4 : 2;
    // How many groups a tile holds.  A workgroup costs about 2 us whatever it holds, and narrow ones read parts of cache lines, so with work for
    // every compute unit the most groups that stay under 96 KB (dx with silu: 1024 x 26 x 26 x 32 fp32 in 8 groups, 86 KB 50 us, 43 KB 52 us, 11 KB
    // 97 us; 64 x 32 x 32 x 256 in 32 groups, 64 KB 38 us, 32 KB 41 us, 8 KB 60 us).  With little work the fewest groups: one sample of 28 x 28 x 32 in 8
    // workgroups 5.8 us, in one 7.5 us.  A tile of more than 96 KB leaves a compute unit with one workgroup that loads, waits and stores in
    // turn: the sample is cut into runs of rows and read twice (48 x 64 x 64 x 512 bfloat16 with silu, held in 32-byte rows: forward 148 us, dx
    // 224 us; cut, with 128-byte rows: 116 and 188 us).
    int best = 0;
    for (int K = 1; K <= G; K = K < G && (K + 1) * p.D > 4 * GROUP_THREADS ? G : K + 1) {
        if (G % K || !widen(p, K)) continue;
        if (p.rows <= GROUP_THREADS / p.TX * most && (int64_t)p.rows * p.TX * 4 * size <= 96 << 10 && (!best || B * (G / K) >= 512)) best = K;
        if (K == G) break;
    }
    if (best) {
        widen(p, best);
        // rows per thread: many amortise what a workgroup costs (the first shape in 43 KB tiles, dx with silu: 8 rows 52 us, 4 rows 72 us), few
        // spread little work over more threads
        held = B * p.chunks >= 512 ? most : 4;
        while ((p.rows + held - 1) / held * p.TX > GROUP_THREADS) held *= 2;
        // The backward pass takes 120 registers: 16 wavefronts per compute unit.  A workgroup of 9 to 11 leaves it no second one to load
        // while the first computes, one of 5 leaves four places empty: where rows kept in LDS bring it down to 8 or 4, two or four
        // fit (1024 x 26 x 26 x 32 in 8 groups, dx with silu: fp32, 11 -> 8, 61 -> 50 us; bfloat16, 2048 samples in 4 groups, 6 -> 4, 86 -> 64 us).  Elsewhere they only
        // cost (1024 x 20 x 20 x 32, 7 -> 5: 38 -> 48 us).
        const int more = most + in_lds(most);
        for (int fits = 512; backward && held == most && p.K <= 512 && fits >= 256; fits /= 2)  // (K: 64 KB hold the rows and the groups' sums)
            if ((p.rows + most - 1) / most * p.TX > fits && (p.rows + more - 1) / more * p.TX <= fits) held = more;
        p.TY = (p.rows + held - 1) / held;
        p.splits = 1, p.split_rows = p.rows;
        const int one = p.TY * p.TX;  // small samples share a workgroup while there are enough of them
        while ((p.NS + 1) * one <= 256 && B / (p.NS + 1) * p.chunks >= 512) ++p.NS;
    } else {
        // rows of 128 bytes or more, whole lines (dx with silu: 48 x 64 x 64 x 512 bfloat16 in 32 groups, 128 bytes 188 us, 64 bytes 213 us, 32 bytes
        // 271 us; 16 x 128 x 128 x 64 fp32 in 8 groups 58, 57 and 61 us)
        for (int K = 1; K <= G; K = K < G && (K + 1) * p.D > 4 * GROUP_THREADS ? G : K + 1) {
            if (G % K == 0 && widen(p, K)) {
                best = K;
                if (p.TX * 4 * size >= 128) break;
            }
            if (K == G) break;
        }
        if (!best) return false;
        widen(p, best);
        held = most;
        p.TY = 256 / p.TX > 1 ? 256 / p.TX : 1;
        p.split_rows = p.TY * held;
        p.splits = (p.rows + p.split_rows - 1) / p.split_rows;
    }
    threads = (p.NS * p.TY * p.TX + 63) / 64 * 64;
    p.team = 1;
    while (p.team < 64 && p.team * 2 * p.NS * p.K <= threads) p.team *= 2;
    const int64_t tiles = (B + p.NS - 1) / p.NS * p.splits;
    if ((tiles + 7) * p.chunks * threads > 0xffffffff) return false;  // (a launch has less than 2^32 threads)
    p.tiles = (int)tiles;
    // What a pass reads and writes against the card's 256 MB cache, and rows of whole lines: 48 x 64 x 64 x 512 bfloat16 with silu, forward 119 -> 116
    // us, dx 192 -> 188 us, before a relu 120 -> 118 and 241 -> 237 us (without an activation 114 -> 122 and 184 -> 183 us).  Half lines are slower
    // that way (64 x 32 x 32 x 256 fp32 in rows of 64 bytes, backward 50 -> 54 us), and a smaller output is still there for the layer
    // that reads it next.
    p.through = B * S * C * size * (backward ? 3 : 2) > (int64_t)256 << 20 && p.TX * 4 * size % 128 == 0;
    return true;
}

// n slices of terms of dgamma and dbeta, and runs of them added up - runs of runs - until the last reduction takes them: it adds n / 128 in a row
int64_t slices_floats(int64_t n, int C) {
    int64_t all = n;
    for (; n > MOST_SLICES; all += n) n = (n + SLICE_RUN - 1) / SLICE_RUN;
    return 2 * (int64_t)C * all;
}

int sum_slices(float *slices, int64_t n, int C, float *dgamma, float *dbeta, hipStream_t st) {
    const int64_t M = 2 * (int64_t)C;
    while (n > MOST_SLICES) {
        const int64_t runs = (n + SLICE_RUN - 1) / SLICE_RUN;
        float *joined = slices + n * M;
        hipLaunchKernelGGL(group_norm_join_slices, dim3((unsigned)((M + 63) / 64), (unsigned)(runs < 65535 ? runs : 65535)), dim3(64), 0, st, slices, n, M, joined);
        const int rc = check_launch("hgq_group_norm_bwd");
        if (rc) return rc;
        slices = joined, n = runs;
    }
    return reduce_parts(slices, (int)n, M, dgamma, C, dbeta, C, nullptr, 0, st);
}

int64_t parts_floats(const GroupTile &p, bool backward) { return p.splits > 1 ? p.B * p.splits * p.G * (backward ? 2 : 4) : 0; }

int lds_bytes(const GroupTile &p, int threads, int held, int type, int act, bool backward) {
    const int most = most_held(type), kept = held > most ? 16 + in_lds(most) * 2 * threads * (type == HGQ_TYPE_F32 ? 16 : 8) : 0;
    const int size = act == HGQ_ACT_RELU && !backward ? 8 : 4;
    return size * (2 * p.NS * p.K + threads * (p.D % 4 == 0 && !backward ? 1 : 4)) + kept;
}

unsigned any_grid(const GroupShape &s) { return (unsigned)(s.B * s.G < 1 << 20 ? s.B * s.G : 1 << 20); }

unsigned blocks(const GroupTile &p) { return (unsigned)(((int64_t)p.tiles + 7) / 8 * 8 * p.chunks); }

template <typename T, int ACT, bool ONE>
auto fwd_kernel(int held) {
    return held == 4 ? group_norm_fwd_tile<T, ACT, ONE, 4> : held == 8 ? group_norm_fwd_tile<T, ACT, ONE, 8> : group_norm_fwd_tile<T, ACT, ONE, MOST_HELD<T>>;
}

template <typename T, int ACT, bool ONE>
auto bwd_kernel(int held) {
    constexpr int most = MOST_HELD<T>;
    return held > most ? group_norm_bwd_tile<T, ACT, ONE, most, in_lds(most)>
           : held == 4 ? group_norm_bwd_tile<T, ACT, ONE, 4, 0>
           : held == 8 ? group_norm_bwd_tile<T, ACT, ONE, 8, 0>
                       : group_norm_bwd_tile<T, ACT, ONE, most, 0>;
}

template <typename T, int ACT>
int fwd(const void *x, const float *gamma, const float *beta, void *y, double *mean, double *rstd, float *ws, const GroupShape &s, int type,
        hipStream_t st) {
    GroupTile p;
    int held, threads;
    if (!plan(p, held, threads, s.B, s.S, s.C, s.G, type, false)) {
        hipLaunchKernelGGL((group_norm_fwd_any<T, ACT>), dim3(any_grid(s)), dim3(256), 0, st, (const T *)x, gamma, beta, (T *)y, mean, rstd, s);
        return check_launch("hgq_group_norm_fwd");
    }
    p.eps = s.eps;
    if (p.splits > 1 && !ws) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: null workspace");
    auto kernel = p.D % 4 == 0 ? fwd_kernel<T, ACT, true>(held) : fwd_kernel<T, ACT, false>(held);
    for (int phase = p.splits > 1 ? 1 : 0; phase < (p.splits > 1 ? 3 : 1); ++phase) {
        hipLaunchKernelGGL(kernel, dim3(blocks(p)), dim3(threads), lds_bytes(p, threads, held, type, ACT, false), st, (const T *)x, gamma, beta, (T *)y, mean, rstd, (double *)ws, p, phase);
        const int rc = check_launch("hgq_group_norm_fwd");
        if (rc) return rc;
    }
    return HGQ_OK;
}

template <typename T, int ACT>
int bwd(const void *dy, const void *x, const float *gamma, const float *beta, const double *mean, const double *rstd, void *dx, float *dgamma,
        float *dbeta, float *ws, const GroupShape &s, int type, hipStream_t st) {
    const bool sums = dgamma || dbeta;
    GroupTile p;
    int held, threads;
    if (!plan(p, held, threads, s.B, s.S, s.C, s.G, type, true)) {
        hipLaunchKernelGGL((group_norm_bwd_any<T, ACT>), dim3(any_grid(s)), dim3(256), 0, st, (const T *)dy, (const T *)x, gamma, beta, mean, rstd, (T *)dx,
                           sums ? ws : nullptr, s);
        const int rc = check_launch("hgq_group_norm_bwd");
        if (rc || !sums) return rc;
        return sum_slices(ws, s.B, s.C, dgamma, dbeta, st);
    }
    float *slices = sums ? ws : nullptr, *parts = p.splits > 1 ? ws + slices_floats(p.tiles, s.C) : nullptr;
    if (p.splits > 1 && !ws) return fail(HGQ_ERR_ARG, "hgq_group_norm_bwd: null workspace");
    auto kernel = p.D % 4 == 0 ? bwd_kernel<T, ACT, true>(held) : bwd_kernel<T, ACT, false>(held);
    for (int phase = p.splits > 1 ? 1 : 0; phase < (p.splits > 1 ? 3 : 1); ++phase) {
        if (phase == 2 && !dx) break;
        hipLaunchKernelGGL(kernel, dim3(blocks(p)), dim3(threads), lds_bytes(p, threads, held, type, ACT, true), st, (const T *)dy, (const T *)x, gamma, beta, mean, rstd,
                           (T *)dx, slices, parts, p, phase);
        const int rc = check_launch("hgq_group_norm_bwd");
        if (rc) return rc;
    }
    return sums ? sum_slices(slices, p.tiles, s.C, dgamma, dbeta, st) : HGQ_OK;
}

template <typename T>
auto fwd_of(int act) {
    return act == HGQ_ACT_RELU ? fwd<T, HGQ_ACT_RELU> : act == HGQ_ACT_SILU ? fwd<T, HGQ_ACT_SILU> : fwd<T, HGQ_ACT_NONE>;
}

template <typename T>
auto bwd_of(int act) {
    return act == HGQ_ACT_RELU ? bwd<T, HGQ_ACT_RELU> : act == HGQ_ACT_SILU ? bwd<T, HGQ_ACT_SILU> : bwd<T, HGQ_ACT_NONE>;
}

}  // namespace

extern "C" int64_t hgq_group_norm_fwd_workspace(int64_t B, int64_t S, int C, int G, int type) {
    if (check_shape("hgq_group_norm_fwd_workspace", B, S, C, G, HGQ_ACT_NONE, type)) return -1;
    GroupTile p;
    int held, threads;
    return plan(p, held, threads, B, S, C, G, type, false) ? parts_floats(p, false) : 0;
}

extern "C" int64_t hgq_group_norm_bwd_workspace(int64_t B, int64_t S, int C, int G, int type) {
    if (check_shape("hgq_group_norm_bwd_workspace", B, S, C, G, HGQ_ACT_NONE, type)) return -1;
    GroupTile p;
    int held, threads;
    return plan(p, held, threads, B, S, C, G, type, true) ? slices_floats(p.tiles, C) + parts_floats(p, true) : slices_floats(B, C);
}

extern "C" int hgq_group_norm_fwd(const void *x, const float *gamma, const float *beta, void *y, double *mean, double *rstd, float *workspace,
                                  int64_t B, int64_t S, int C, int G, float eps, int act, int type, void *stream) {
    int rc = check_shape("hgq_group_norm_fwd", B, S, C, G, act, type);
    if (rc) return rc;
    if (!(eps >= 0)) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: epsilon must not be negative");
    if (B == 0 || S == 0) return HGQ_OK;
    if (!x || !y || !mean || !rstd) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: null pointer");
    const GroupShape s = {B, S, C, G, C / G, eps};
    return (type == HGQ_TYPE_F32 ? fwd_of<float>(act) : type == HGQ_TYPE_BF16 ? fwd_of<__bf16>(act) : fwd_of<_Float16>(act))(x, gamma, beta, y, mean, rstd, workspace, s, type, (hipStream_t)stream);
}

extern "C" int hgq_group_norm_bwd(const void *dy, const void *x, const float *gamma, const float *beta, const double *mean, const double *rstd,
                                  void *dx, float *dgamma, float *dbeta, float *workspace, int64_t B, int64_t S, int C, int G, int act, int type,
                                  void *stream) {
    int rc = check_shape("hgq_group_norm_bwd", B, S, C, G, act, type);
    if (rc) return rc;
    if (B == 0 || S == 0) {
        if (dgamma && (rc = fill_f32(dgamma, 0.0f, C, (hipStream_t)stream))) return rc;
        return dbeta ? fill_f32(dbeta, 0.0f, C, (hipStream_t)stream) : HGQ_OK;
    }
    if (!dy || !x || !mean || !rstd || ((dgamma || dbeta) && !workspace)) return fail(HGQ_ERR_ARG, "hgq_group_norm_bwd: null pointer");
    if (!dx && !dgamma && !dbeta) return HGQ_OK;
    const GroupShape s = {B, S, C, G, C / G, 0.0f};
    return (type == HGQ_TYPE_F32 ? bwd_of<float>(act) : type == HGQ_TYPE_BF16 ? bwd_of<__bf16>(act) : bwd_of<_Float16>(act))(dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, workspace, s,
                                                                                                    type, (hipStream_t)stream);
}
