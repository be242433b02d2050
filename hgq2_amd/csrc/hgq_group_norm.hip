// Group normalisation with an activation over channels-last tensors x [B, S, C], S positions, C = G D channels in G groups:
//     mean, var over the S D elements of a sample's group;   xhat = (x - mean) / sqrt(var + eps)
//     z = xhat gamma[c] + beta[c];   y = act(z)
// Backward, with dz = dy act'(z) and d = dz gamma:
//     dx = (d - mean(d) - xhat mean(d xhat)) / sqrt(var + eps);   dgamma[c] = sum dz xhat,  dbeta[c] = sum dz  over B and S
// x, y, dy and dx have one of three types; everything between is fp32, the variance about the mean (not a difference of squares).
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

// z of d = x - mean.  Before a relu the roundings follow the formula's order, (d rstd) gamma + beta: which side of zero a value falls on that
// lies within rounding of it is then the same for every program that does so with the same mean (11 of 160 tensors of 22 million elements held
// one that fell differently from an fp32 evaluation by elementary operations; 13 of 120 with d (rstd gamma) + beta in one rounding).
template <int ACT>
__device__ __forceinline__ float affine(float d, float rstd, float gamma, float scale, float beta) {
    if (ACT == HGQ_ACT_RELU) return __fadd_rn(__fmul_rn(__fmul_rn(d, rstd), gamma), beta);
    return fmaf(d, scale, beta);  // scale: rstd gamma
}

// dy act'(z)
template <int ACT>
__device__ __forceinline__ float through_activation(float dy, float z) {
    if (ACT == HGQ_ACT_RELU) return z > 0.0f ? dy : z != z ? z : 0.0f;
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
                                                          T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out, GroupShape s) {
    __shared__ double lds[4];
    for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
        const int64_t b = bg / s.G;
        const int g = (int)(bg - b * s.G);
        const int64_t base = b * s.S * s.C + (int64_t)g * s.D, n = s.S * s.D;
        double sum = 0;
        for (int64_t e = threadIdx.x; e < n; e += 256) sum += to_f32(x[base + e / s.D * s.C + e % s.D]);
        const float mean = (float)(group_sum(sum, lds) / (double)n);
        double sq = 0;
        for (int64_t e = threadIdx.x; e < n; e += 256) {
            const float d = to_f32(x[base + e / s.D * s.C + e % s.D]) - mean;
            sq += (double)d * d;
        }
        const float rstd = 1.0f / sqrtf((float)(group_sum(sq, lds) / (double)n) + s.eps);
        if (threadIdx.x == 0) mean_out[bg] = mean, rstd_out[bg] = rstd;
        for (int64_t e = threadIdx.x; e < n; e += 256) {
            const int c = g * s.D + (int)(e % s.D);
            const int64_t at = base + e / s.D * s.C + e % s.D;
            const float ga = gamma ? gamma[c] : 1.0f, z = affine<ACT>(to_f32(x[at]) - mean, rstd, ga, rstd * ga, beta ? beta[c] : 0.0f);
            y[at] = (T)activate<ACT>(z);
        }
    }
}

// A workgroup takes one sample's group after another, any shape.  part [B][2 C]: each sample's terms of dgamma, then of dbeta.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void group_norm_bwd_any(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                          const float *__restrict__ beta, const float *__restrict__ mean_in,
                                                          const float *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ part, GroupShape s) {
    __shared__ double lds[4];
    __shared__ double col[2][256];
    int tx = 1;  // threads side by side over channels, the others over positions
    while (tx < s.D && tx < 256) tx *= 2;
    const int ty = 256 / tx, cx = threadIdx.x % tx, py = threadIdx.x / tx;
    for (int64_t bg = blockIdx.x; bg < s.B * s.G; bg += gridDim.x) {
        const int64_t b = bg / s.G;
        const int g = (int)(bg - b * s.G);
        const int64_t base = b * s.S * s.C + (int64_t)g * s.D, n = s.S * s.D;
        const float mean = mean_in[bg], rstd = rstd_in[bg];
        double s1 = 0, s2 = 0;  // of d and d xhat, over the group
        for (int c0 = 0; c0 < s.D; c0 += tx) {
            const int d = c0 + cx, c = g * s.D + d;
            double a = 0, h = 0;
            const float ga = d < s.D && gamma ? gamma[c] : 1.0f, be = d < s.D && beta ? beta[c] : 0.0f;
            if (d < s.D)
                for (int64_t p = py; p < s.S; p += ty) {
                    const int64_t at = base + p * s.C + d;
                    const float xh = (to_f32(x[at]) - mean) * rstd;
                    const float dz = through_activation<ACT>(to_f32(dy[at]), xh * ga + be);
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
            const float ga = gamma ? gamma[c] : 1.0f, xh = (to_f32(x[at]) - mean) * rstd;
            const float dz = through_activation<ACT>(to_f32(dy[at]), xh * ga + (beta ? beta[c] : 0.0f));
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
template <bool ONE>
__device__ __forceinline__ void sum_groups(const GroupTile &p, const GroupThread &t, const float (&v)[4], float *red, float *total) {
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
        const float *mine = red + (g / p.K) * p.TY * width + (g % p.K) * across;
        float sum = 0;
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
                                                            T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out,
                                                            float *__restrict__ parts, GroupTile p, int phase) {
    extern __shared__ float lds[];
    const int groups = p.NS * p.K;
    float *total = lds, *stat = lds + groups, *red = lds + 2 * groups;
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
    if (phase < 2) {
        float acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += v[i].get(j);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) acc[j] += last[j];
        sum_groups<ONE>(p, t, acc, red, total);
        // elements of a group in this tile
        const float inv = p.splits == 1 ? p.inv : 1.0f / (float)((min(p.n / p.C, r1 * p.fold) - r0 * p.fold) * p.D);
#pragma unroll
        for (int j = 0; j < N; ++j) mean[j] = t.on ? total[group_of<ONE>(p, t, j)] * inv : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < rows.full) {
                v[i].forget();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float d = v[i].get(j) - mean[j % N];
                    acc[j] = fmaf(d, d, acc[j]);
                }
            }
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < rows.rest) {
                const float d = last[j] - mean[j % N];
                acc[j] = fmaf(d, d, acc[j]);
            }
        sum_groups<ONE>(p, t, acc, red, stat);
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            const int64_t bg = z / p.splits * p.NS + g / p.K;
            if (bg >= p.B) break;
            const int64_t at = bg * p.G + chunk * p.K + g % p.K;
            if (phase == 1) {
                float *out = parts + ((bg * p.splits + split) * p.G + chunk * p.K + g % p.K) * 2;
                out[0] = total[g] * inv, out[1] = stat[g];
            } else {
                mean_out[at] = total[g] * inv, rstd_out[at] = 1.0f / sqrtf(stat[g] * p.inv + p.eps);
            }
        }
        if (phase == 1) return;
#pragma unroll
        for (int j = 0; j < N; ++j) rstd[j] = t.on ? 1.0f / sqrtf(stat[group_of<ONE>(p, t, j)] * p.inv + p.eps) : 0.0f;
    } else {
        // the splits' means about the first one's, and their squares about the joint mean
        const int lane = threadIdx.x & (p.team - 1);
        for (int g = threadIdx.x / p.team; g < groups; g += blockDim.x / p.team) {
            const float *in = parts + (b - t.s) * p.splits * p.G * 2 + (chunk * p.K + g) * 2;  // (one sample: NS = 1)
            const float first = in[0];
            float m = 0, q = 0;
            for (int k = lane; k < p.splits; k += p.team) {
                const float w = (float)((min(p.n / p.C, (k + 1) * p.split_rows * p.fold) - k * p.split_rows * p.fold) * p.D) * p.inv;
                m += w * (in[(int64_t)k * p.G * 2] - first);
            }
            for (int d = p.team / 2; d; d >>= 1) m += __shfl_xor(m, d);
            for (int k = lane; k < p.splits; k += p.team) {
                const float w = (float)((min(p.n / p.C, (k + 1) * p.split_rows * p.fold) - k * p.split_rows * p.fold) * p.D) * p.inv;
                const float d = in[(int64_t)k * p.G * 2] - first - m;
                q += in[(int64_t)k * p.G * 2 + 1] * p.inv + w * d * d;
            }
            for (int d = p.team / 2; d; d >>= 1) q += __shfl_xor(q, d);
            if (lane == 0) {
                total[g] = first + m, stat[g] = 1.0f / sqrtf(q + p.eps);
                if (split == 0) mean_out[(b - t.s) * p.G + chunk * p.K + g] = total[g], rstd_out[(b - t.s) * p.G + chunk * p.K + g] = stat[g];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) mean[j] = t.on ? total[group_of<ONE>(p, t, j)] : 0.0f, rstd[j] = t.on ? stat[group_of<ONE>(p, t, j)] : 0.0f;
    }
    if (!on) return;
    float ga[4], scale[4], be[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = p.fold > 1 ? (c0 + j) % p.C : c0 + j;
        ga[j] = gamma ? gamma[c] : 1.0f, scale[j] = rstd[j % N] * ga[j], be[j] = beta ? beta[c] : 0.0f;
    }
    T *ys = y + b * p.n;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i < rows.full) {
            v[i].forget();
            float out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = activate<ACT>(affine<ACT>(v[i].get(j) - mean[j % N], rstd[j % N], ga[j], scale[j], be[j]));
            v[i].set(out);
            v[i].store(ys + rows.at + i * rows.step, p.through);
        }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < rows.rest) ys[rows.at + rows.full * rows.step + j] = (T)activate<ACT>(affine<ACT>(last[j] - mean[j % N], rstd[j % N], ga[j], scale[j], be[j]));
}

// phase 0: whole tiles; 1: sums of d rstd and d xhat rstd of every split, parts [B][splits][G][2], and the channels' sums; 2: join them, dx.
// Every tile leaves its terms of dgamma and dbeta, slices [tiles][2 C] (NULL: not wanted).  MORE: rows of a thread beyond those in its registers, which it
// keeps in LDS.
template <typename T, int ACT, bool ONE, int NV, int MORE>
__global__ __launch_bounds__(MORE ? 512 : 1024, 4) void group_norm_bwd_tile(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                            const float *__restrict__ beta, const float *__restrict__ mean_in,
                                                            const float *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ slices,
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
    float mean[N], rstd[N], ga[4], scale[4], be[4];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int64_t g = b * p.G + chunk * p.K + group_of<ONE>(p, t, j) - t.s * p.K;
        mean[j] = on ? mean_in[g] : 0.0f, rstd[j] = on ? rstd_in[g] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = p.fold > 1 ? (c0 + j) % p.C : c0 + j;
        ga[j] = t.on && gamma ? gamma[c] : 1.0f, scale[j] = rstd[j % N] * ga[j], be[j] = t.on && beta ? beta[c] : 0.0f;
    }
    // rstd gamma: before a relu the two are needed by themselves, and their product is not kept beside them
    auto times = [&](int j) { return ACT == HGQ_ACT_RELU ? rstd[j % N] * ga[j] : scale[j]; };
    float h[4] = {0, 0, 0, 0}, a[4] = {0, 0, 0, 0};  // of dz (x - mean) and of dz
    if (phase < 2) {
        float mine[2][4];
        auto add = [&](float xv, float dv, int j) {
            const float d = xv - mean[j % N], dz = through_activation<ACT>(dv, affine<ACT>(d, rstd[j % N], ga[j], scale[j], be[j]));
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
            float m1 = 0, m2 = 0;
            for (int k = lane; k < p.splits; k += p.team) m1 += in[(int64_t)k * p.G * 2], m2 += in[(int64_t)k * p.G * 2 + 1];
            for (int d = p.team / 2; d; d >>= 1) m1 += __shfl_xor(m1, d), m2 += __shfl_xor(m2, d);
            if (lane == 0) total[g] = m1, stat[g] = m2;
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
            const float d = xv - mean[j % N], dz = through_activation<ACT>(dv, affine<ACT>(d, rstd[j % N], ga[j], scale[j], be[j]));
            return fmaf(dz, times(j), fmaf(d, m2[j % N], m1[j % N]));
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
    const int width = p.TX * 4, cols = p.K * p.D, folds = p.fold == 4 ? 2 : p.fold - 1, count = (p.NS * p.TY) << folds;  // (fold = 1, 2 or 4)
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
    // How many groups a tile holds.  A workgroup costs about 2 us whatever it holds, so with work for every compute unit the most groups that
    // stay under 96 KB (1024 x 26 x 26 x 32 fp32 in 8 groups, backward: 86 KB 68 us, 43 KB 74 us, 11 KB 97 us; 256 x 8 x 8 x 512: 64 KB 22 us, 4 KB 29 us).
    // With little work the fewest groups: one sample of 28 x 28 x 32 in 8 workgroups 5.8 us, in one 7.5 us.  A tile of more than 96 KB
    // leaves a compute unit with one workgroup that loads, waits and stores in turn, and narrow ones read parts of cache lines: the
    // sample is cut into runs of rows and read twice (48 x 64 x 64 x 512 bfloat16: held, 32-byte rows 148 us, cut with 128-byte rows 127 us).
    int best = 0;
    for (int K = 1; K <= G; K = K < G && (K + 1) * p.D > 4 * GROUP_THREADS ? G : K + 1) {
        if (G % K || !widen(p, K)) continue;
        if (p.rows <= GROUP_THREADS / p.TX * most && (int64_t)p.rows * p.TX * 4 * size <= 96 << 10 && (!best || B * (G / K) >= 512)) best = K;
        if (K == G) break;
    }
    if (best) {
        widen(p, best);
        // rows per thread: many amortise what a workgroup costs (the first shape in 43 KB tiles, backward: 8 rows 74 us, 4 rows 97 us), few
        // spread little work over more threads
        held = B * p.chunks >= 512 ? most : 4;
        while ((p.rows + held - 1) / held * p.TX > GROUP_THREADS) held *= 2;
        // The backward pass takes 120 registers: 16 wavefronts per compute unit.  A workgroup of 9 to 11 leaves it no second one to load
        // while the first computes, one of 5 leaves four places empty: where rows kept in LDS bring it down to 8 or 4, two or four
        // fit (1024 x 26 x 26 x 32 in 8 groups: fp32, 11 -> 8, 70 -> 54 us; bfloat16, 2048 samples in 4 groups, 6 -> 4, 98 -> 63 us).  Elsewhere they only
        // cost (1024 x 20 x 20 x 32, 7 -> 5: 38 -> 48 us).
        const int more = most + in_lds(most);
        for (int fits = 512; backward && held == most && fits >= 256; fits /= 2)
            if ((p.rows + most - 1) / most * p.TX > fits && (p.rows + more - 1) / more * p.TX <= fits) held = more;
        p.TY = (p.rows + held - 1) / held;
        p.splits = 1, p.split_rows = p.rows;
        const int one = p.TY * p.TX;  // small samples share a workgroup while there are enough of them
        while ((p.NS + 1) * one <= 256 && B / (p.NS + 1) * p.chunks >= 512) ++p.NS;
    } else {
        // rows of 128 bytes or more, whole lines (16 x 128 x 128 x 64 fp32 in 8 groups, backward: 128 bytes 59 us, 32 bytes and less over 63 us)
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
    // What a pass reads and writes against the card's 256 MB cache, and rows of whole lines: 48 x 64 x 64 x 512 bfloat16, forward 131 -> 110 us,
    // backward 206 -> 196 us, and 7 and 6 us less with the second read of its cut samples past the cache as well.  Half lines are slower
    // that way (64 x 32 x 32 x 256 fp32 in rows of 64 bytes, backward 50 -> 54 us), and a smaller output is still there for the layer
    // that reads it next.
    p.through = B * S * C * size * (backward ? 3 : 2) > (int64_t)256 << 20 && p.TX * 4 * size % 128 == 0;
    return true;
}

// the tiles' terms of dgamma and dbeta, and runs of them added up where they are many
int64_t slices_floats(const GroupTile &p) { return 2 * (int64_t)p.C * (p.tiles + (p.tiles > MOST_SLICES ? (p.tiles + SLICE_RUN - 1) / SLICE_RUN : 0)); }

int64_t parts_floats(const GroupTile &p) { return p.splits > 1 ? p.B * p.splits * p.G * 2 : 0; }

int lds_bytes(const GroupTile &p, int threads, int held, int type, bool backward) {
    const int most = most_held(type), kept = held > most ? 16 + in_lds(most) * 2 * threads * (type == HGQ_TYPE_F32 ? 16 : 8) : 0;
    return 4 * (2 * p.NS * p.K + threads * (p.D % 4 == 0 && !backward ? 1 : 4)) + kept;
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
int fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, float *ws, const GroupShape &s, int type,
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
        hipLaunchKernelGGL(kernel, dim3(blocks(p)), dim3(threads), lds_bytes(p, threads, held, type, false), st, (const T *)x, gamma, beta, (T *)y, mean, rstd, ws, p, phase);
        const int rc = check_launch("hgq_group_norm_fwd");
        if (rc) return rc;
    }
    return HGQ_OK;
}

template <typename T, int ACT>
int bwd(const void *dy, const void *x, const float *gamma, const float *beta, const float *mean, const float *rstd, void *dx, float *dgamma,
        float *dbeta, float *ws, const GroupShape &s, int type, hipStream_t st) {
    const bool sums = dgamma || dbeta;
    GroupTile p;
    int held, threads;
    if (!plan(p, held, threads, s.B, s.S, s.C, s.G, type, true)) {
        hipLaunchKernelGGL((group_norm_bwd_any<T, ACT>), dim3(any_grid(s)), dim3(256), 0, st, (const T *)dy, (const T *)x, gamma, beta, mean, rstd, (T *)dx,
                           sums ? ws : nullptr, s);
        const int rc = check_launch("hgq_group_norm_bwd");
        if (rc || !sums) return rc;
        return reduce_parts(ws, (int)s.B, 2 * (int64_t)s.C, dgamma, s.C, dbeta, s.C, nullptr, 0, st);
    }
    const int64_t M = 2 * (int64_t)s.C;
    float *slices = sums ? ws : nullptr, *parts = p.splits > 1 ? ws + slices_floats(p) : nullptr;
    if (p.splits > 1 && !ws) return fail(HGQ_ERR_ARG, "hgq_group_norm_bwd: null workspace");
    auto kernel = p.D % 4 == 0 ? bwd_kernel<T, ACT, true>(held) : bwd_kernel<T, ACT, false>(held);
    for (int phase = p.splits > 1 ? 1 : 0; phase < (p.splits > 1 ? 3 : 1); ++phase) {
        if (phase == 2 && !dx) break;
        hipLaunchKernelGGL(kernel, dim3(blocks(p)), dim3(threads), lds_bytes(p, threads, held, type, true), st, (const T *)dy, (const T *)x, gamma, beta, mean, rstd,
                           (T *)dx, slices, parts, p, phase);
        const int rc = check_launch("hgq_group_norm_bwd");
        if (rc) return rc;
    }
    if (!sums) return HGQ_OK;
    if (p.tiles <= MOST_SLICES) return reduce_parts(slices, p.tiles, M, dgamma, s.C, dbeta, s.C, nullptr, 0, st);
    const int runs = (p.tiles + SLICE_RUN - 1) / SLICE_RUN;
    float *joined = slices + p.tiles * M;
    hipLaunchKernelGGL(group_norm_join_slices, dim3((unsigned)((M + 63) / 64), (unsigned)(runs < 65535 ? runs : 65535)), dim3(64), 0, st, slices, (int64_t)p.tiles, M, joined);
    const int rc = check_launch("hgq_group_norm_bwd");
    return rc ? rc : reduce_parts(joined, runs, M, dgamma, s.C, dbeta, s.C, nullptr, 0, st);
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
    return plan(p, held, threads, B, S, C, G, type, false) ? parts_floats(p) : 0;
}

extern "C" int64_t hgq_group_norm_bwd_workspace(int64_t B, int64_t S, int C, int G, int type) {
    if (check_shape("hgq_group_norm_bwd_workspace", B, S, C, G, HGQ_ACT_NONE, type)) return -1;
    GroupTile p;
    int held, threads;
    return plan(p, held, threads, B, S, C, G, type, true) ? slices_floats(p) + parts_floats(p) : B * 2 * C;
}

extern "C" int hgq_group_norm_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, float *workspace,
                                  int64_t B, int64_t S, int C, int G, float eps, int act, int type, void *stream) {
    int rc = check_shape("hgq_group_norm_fwd", B, S, C, G, act, type);
    if (rc) return rc;
    if (!(eps >= 0)) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: epsilon must not be negative");
    if (B == 0 || S == 0) return HGQ_OK;
    if (!x || !y || !mean || !rstd) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: null pointer");
    const GroupShape s = {B, S, C, G, C / G, eps};
    return (type == HGQ_TYPE_F32 ? fwd_of<float>(act) : type == HGQ_TYPE_BF16 ? fwd_of<__bf16>(act) : fwd_of<_Float16>(act))(x, gamma, beta, y, mean, rstd, workspace, s, type, (hipStream_t)stream);
}

extern "C" int hgq_group_norm_bwd(const void *dy, const void *x, const float *gamma, const float *beta, const float *mean, const float *rstd,
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
