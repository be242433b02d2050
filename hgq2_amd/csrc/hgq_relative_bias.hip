// A learned bias by relative position on attention scores [B, H, T, S], and its gradient:
//     out[b, h, i, j] = scores[b, h, i, j] + table[bucket(d), h],   d = j - (i + offset),   n buckets, m = n (or n / 2, two-sided) a direction
//     bucket = how many of the first distances of buckets 1 .. m - 1 lie at or below |d| (one-sided: max(-d, 0)), plus m for d > 0 (two-sided)
//     dtable[k, h] = sum of dscores over all b, i, j with bucket(d) = k;   the gradient of the scores is that of the output
// Both are bound by memory: scores in, out out; the gradient is read once.  The T S elements of a (b, h) lie one after the other, so a
// thread takes 16 bytes of them at any row length, and keeps them for a run of the batch: what the position costs (a division, the buckets) is paid once
// per thread in the forward pass, and the gradient's terms meet in registers over the batch before they meet over buckets.  There each lane has bins
// of its own in LDS (no atomics: sums have an order), and neighbouring elements of one bucket, all but those near the diagonal, are
// added before they are put in.
#include "hgq_host.h"
#include "hgq_vector.h"

namespace hgq {

constexpr int BIAS_BUCKETS = 128;
constexpr int BIAS_NEAR = 4096;  // distances whose bucket a workgroup looks up; beyond, where buckets still change there, it searches

struct BiasShape {
    int first[BIAS_BUCKETS];  // of buckets 1 .. m - 1
    int64_t stride_b, stride_h, offset;
    const void *offsets;  // [B] (int32 or int64) or null
    int B, H, S, TS, m, both, wide, near, chunk, chunks, tiles;
};

__device__ __forceinline__ int bucket_of(const BiasShape &s, const int *first, int d) {
    const int n = s.both ? abs(d) : max(-d, 0);
    int lo = 0, hi = s.m - 1;  // how many first distances are <= n
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= n) lo = mid + 1;
        else hi = mid;
    }
    return lo + (s.both && d > 0 ? s.m : 0);
}

// distance of element e of the plane, held within what an int's arithmetic takes
__device__ __forceinline__ int distance(int i, int j, int64_t offset) {
    const int64_t d = (int64_t)j - i - offset;
    return (int)(d < -(1 << 30) ? -(1 << 30) : d > 1 << 30 ? 1 << 30 : d);
}

__device__ __forceinline__ int64_t offset_of(const BiasShape &s, int b) {
    return !s.offsets ? s.offset : s.wide ? ((const int64_t *)s.offsets)[b] : (int64_t)((const int32_t *)s.offsets)[b];
}

// Workgroup: 256 threads, one access each; blocks run over tiles of the plane, heads and runs of the batch.
template <typename T>
__global__ __launch_bounds__(256) void relative_bias_add(const T *__restrict__ scores, const float *__restrict__ table, T *__restrict__ out, const BiasShape s) {
    constexpr int N = Vec<T>::N, AHEAD = 4;
    extern __shared__ float by_distance[];  // [2 near + 1], then the first distances
    int *first = (int *)(by_distance + 2 * s.near + 1);
    for (int k = threadIdx.x; k < s.m - 1; k += 256) first[k] = s.first[k];
    __syncthreads();
    int block = blockIdx.x;
    const int tile = block % s.tiles;
    block /= s.tiles;
    const int h = block % s.H, b0 = block / s.H * s.chunk, b1 = min(s.B, b0 + s.chunk);
    for (int k = threadIdx.x; k <= 2 * s.near; k += 256) by_distance[k] = table[bucket_of(s, first, k - s.near) * s.H + h];
    __syncthreads();
    const int e0 = (tile * 256 + (int)threadIdx.x) * N;
    if (e0 >= s.TS) return;
    const int i0 = e0 / s.S, j0 = e0 - i0 * s.S, n = min(N, s.TS - e0);
    const bool beyond = s.first[s.m - 2] > s.near;
    float bias[N];
    const T *from = scores + b0 * s.stride_b + h * s.stride_h + e0;
    T *to = out + ((int64_t)b0 * s.H + h) * s.TS + e0;
    const int64_t step = (int64_t)s.H * s.TS;
    for (int b = b0; b < b1; b += AHEAD) {
        Vec<T> v[AHEAD];
        if (n == N) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (b + a < b1) v[a] = load_vec(from + a * s.stride_b);
        } else {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (b + a < b1) v[a] = load_part(from + a * s.stride_b, n, (T)0.0f);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (b + a >= b1) break;
            if (b + a == b0 || s.offsets) {
                const int64_t offset = offset_of(s, b + a);
                int i = i0, j = j0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int d = distance(i, j, offset);
                    bias[e] = beyond && abs(d) > s.near ? table[bucket_of(s, first, d) * s.H + h] : by_distance[max(-s.near, min(s.near, d)) + s.near];
                    if (++j == s.S) j = 0, ++i;
                }
            }
#pragma unroll
            for (int e = 0; e < N; ++e) v[a].v[e] = (T)((float)v[a].v[e] + bias[e]);
            if (n == N) store_vec(to + a * step, v[a]);
            else store_part(to + a * step, v[a], n);
        }
        from += AHEAD * s.stride_b, to += AHEAD * step;
    }
}

// bins [n][threads] of a workgroup: every thread's own
struct BiasRun {
    double *bins;
    int threads, bucket;
    double sum;
    __device__ __forceinline__ void flush() {
        if (bucket >= 0) bins[bucket * threads + threadIdx.x] += sum;
    }
    __device__ __forceinline__ void add(int k, double v) {
        if (k != bucket) flush(), bucket = k, sum = v;
        else sum += v;
    }
};

// Workgroup w of a head takes items w, w + parts, ... - an item: a tile of the plane and a run of the batch.  parts [H][parts][n].
template <typename T>
__global__ __launch_bounds__(256) void relative_bias_sums(const T *__restrict__ dy, double *__restrict__ part, int parts, const BiasShape s) {
    constexpr int N = Vec<T>::N, AHEAD = 8;
    extern __shared__ double bias_lds[];
    const int n_buckets = s.both ? 2 * s.m : s.m, threads = blockDim.x;
    int *first = (int *)(bias_lds + n_buckets * threads);
    uint8_t *near = (uint8_t *)(first + BIAS_BUCKETS);
    for (int k = threadIdx.x; k < s.m - 1; k += threads) first[k] = s.first[k];
    for (int k = threadIdx.x; k < n_buckets * threads; k += threads) bias_lds[k] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k <= 2 * s.near; k += threads) near[k] = (uint8_t)bucket_of(s, first, k - s.near);
    __syncthreads();
    const bool beyond = s.first[s.m - 2] > s.near;
    const int h = blockIdx.x / parts, w = blockIdx.x - h * parts;
    BiasRun run = {bias_lds, threads, -1, 0.0};
    for (int64_t item = w; item < (int64_t)s.tiles * s.chunks; item += parts) {
        const int c = (int)(item / s.tiles), tile = (int)(item - (int64_t)c * s.tiles);
        const int b0 = c * s.chunk, b1 = min(s.B, b0 + s.chunk), e0 = (tile * threads + (int)threadIdx.x) * N;
        if (e0 >= s.TS) continue;
        const int i0 = e0 / s.S, j0 = e0 - i0 * s.S, n = min(N, s.TS - e0);
        const T *from = dy + b0 * s.stride_b + h * s.stride_h + e0;
        double sum[N] = {};
        for (int b = b0; b < b1; b += AHEAD) {  // eight terms pairwise in fp32, their sums in fp64
            Vec<T> v[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (b + a < b1) v[a] = n == N ? load_vec(from + a * s.stride_b) : load_part(from + a * s.stride_b, n, (T)0.0f);
                else {
#pragma unroll
                    for (int e = 0; e < N; ++e) v[a].v[e] = (T)0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float f[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) f[a] = (float)v[a].v[e];
#pragma unroll
                for (int k = AHEAD / 2; k; k /= 2)
#pragma unroll
                    for (int a = 0; a < k; ++a) f[a] += f[a + k];
                sum[e] += f[0];
            }
            from += AHEAD * s.stride_b;
        }
        const int64_t offset = offset_of(s, b0);  // (with offsets of their own, runs are of one sequence)
        auto bucket = [&](int d) { return beyond && abs(d) > s.near ? bucket_of(s, first, d) : (int)near[max(-s.near, min(s.near, d)) + s.near]; };
        const int d0 = distance(i0, j0, offset), k0 = bucket(d0);
        if (n == N && j0 + N <= s.S && bucket(distance(i0, j0 + N - 1, offset)) == k0) {
#pragma unroll
            for (int k = N / 2; k; k /= 2)
#pragma unroll
                for (int e = 0; e < k; ++e) sum[e] += sum[e + k];
            run.add(k0, sum[0]);
        } else {
            int i = i0, j = j0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (e < n) run.add(bucket(distance(i, j, offset)), sum[e]);
                if (++j == s.S) j = 0, ++i;
            }
        }
    }
    run.flush();
    __syncthreads();
    for (int k = threadIdx.x >> 6; k < n_buckets; k += threads >> 6) {
        double v = 0;
        for (int t = threadIdx.x & 63; t < threads; t += 64) v += bias_lds[k * threads + t];
        v = team_sum(v, 64);
        if ((threadIdx.x & 63) == 0) part[(int64_t)blockIdx.x * n_buckets + k] = v;
    }
}

// dtable [n, H] from [H][parts][n]: a wavefront for each of its elements
__global__ __launch_bounds__(256) void relative_bias_join(const double *__restrict__ part, int parts, float *__restrict__ dtable, int n, int H) {
    const int at = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (at >= n * H) return;
    const int k = at / H, h = at - k * H;
    double v = 0;
    for (int p = lane; p < parts; p += 64) v += part[((int64_t)h * parts + p) * n + k];
    v = team_sum(v, 64);
    if (lane == 0) dtable[at] = (float)v;
}

namespace {

int check_bias(const char *what, int64_t B, int64_t H, int64_t T, int64_t S, const int *first, int m, int both, int type, int offset_bytes) {
    if (B < 0 || H < 0 || T < 0 || S < 0 || (offset_bytes != 4 && offset_bytes != 8)) return fail(HGQ_ERR_ARG, "%s: bad shape", what);
    if (type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16) return fail(HGQ_ERR_ARG, "%s: unknown type", what);
    if (m < 2 || !first) return fail(HGQ_ERR_ARG, "%s: %d buckets a direction", what, m);
    if ((both ? 2 : 1) * (int64_t)m > BIAS_BUCKETS) return fail(HGQ_ERR_UNSUPPORTED, "%s: more than %d buckets", what, BIAS_BUCKETS);
    for (int k = 0; k + 1 < m; ++k)
        if (first[k] < 1 || (k && first[k] < first[k - 1]) || first[k] > 1 << 30) return fail(HGQ_ERR_ARG, "%s: first distances of buckets must rise from 1 on, up to 2^30", what);
    if (B > INT32_MAX || H > 1 << 20 || T > INT32_MAX || S > INT32_MAX || T * S > INT32_MAX - (1 << 16)) return fail(HGQ_ERR_UNSUPPORTED, "%s: %lld x %lld positions", what, (long long)T, (long long)S);
    return HGQ_OK;
}

BiasShape bias_shape(int64_t B, int64_t H, int64_t T, int64_t S, const int *first, int m, int both, int64_t offset, const void *offsets, int offset_bytes,
                     int64_t stride_b, int64_t stride_h) {
    BiasShape s = {};
    for (int k = 0; k + 1 < m; ++k) s.first[k] = first[k];
    s.B = (int)B, s.H = (int)H, s.S = (int)S, s.TS = (int)(T * S), s.m = m, s.both = both, s.offset = offset, s.offsets = offsets, s.wide = offset_bytes == 8;
    s.stride_b = stride_b, s.stride_h = stride_h;
    s.near = first[m - 2] < BIAS_NEAR ? first[m - 2] : BIAS_NEAR;
    return s;
}

void cut(BiasShape &s, int64_t threads, int N, int64_t wanted) {  // tiles of the plane, and runs of the batch for `wanted` workgroups
    s.tiles = (int)((s.TS + threads * N - 1) / (threads * N));
    int64_t chunks = s.offsets ? s.B : (wanted + (int64_t)s.tiles * s.H - 1) / ((int64_t)s.tiles * s.H);
    if (chunks > s.B) chunks = s.B;
    s.chunk = (int)((s.B + chunks - 1) / chunks);
    s.chunks = (s.B + s.chunk - 1) / s.chunk;
}

int sums_threads(int n) { return n <= 16 ? 256 : n <= 32 ? 128 : 64; }  // 32 KB of bins up to 64 buckets: five workgroups a compute unit

int sums_parts(const BiasShape &s, int threads) {
    const int64_t items = (int64_t)s.tiles * s.chunks;
    int64_t parts = (512 * (256 / threads) + s.H - 1) / s.H;
    return (int)(items < parts ? items : parts);
}

template <typename T>
int add(const void *scores, const float *table, void *out, BiasShape s, hipStream_t st) {
    cut(s, 256, Vec<T>::N, 2048);
    const int64_t blocks = (int64_t)s.tiles * s.H * s.chunks;
    if (blocks * 256 > 0xffffffffLL) return fail(HGQ_ERR_UNSUPPORTED, "hgq_relative_bias_fwd: too many scores");
    hipLaunchKernelGGL(relative_bias_add<T>, dim3((unsigned)blocks), dim3(256), 4 * (2 * s.near + 1 + BIAS_BUCKETS), st, (const T *)scores, table, (T *)out, s);
    return check_launch("hgq_relative_bias_fwd");
}

template <typename T>
int sums(const void *dy, float *dtable, double *part, BiasShape s, hipStream_t st) {
    const int n = s.both ? 2 * s.m : s.m, threads = sums_threads(n);
    cut(s, threads, Vec<T>::N, 1024);
    const int parts = sums_parts(s, threads);
    const int lds = 8 * n * threads + 4 * BIAS_BUCKETS + 2 * s.near + 1;
    // (more than 112 buckets; per device, so it is asked for at every such call)
    if (lds > 64 << 10 && hipFuncSetAttribute((const void *)relative_bias_sums<T>, hipFuncAttributeMaxDynamicSharedMemorySize, 80 << 10) != hipSuccess) {
        (void)hipGetLastError();
        return fail(HGQ_ERR_LAUNCH, "hgq_relative_bias_bwd: cannot reserve LDS");
    }
    hipLaunchKernelGGL(relative_bias_sums<T>, dim3((unsigned)(parts * s.H)), dim3(threads), lds, st, (const T *)dy, part, parts, s);
    int rc = check_launch("hgq_relative_bias_bwd");
    if (rc) return rc;
    hipLaunchKernelGGL(relative_bias_join, dim3((unsigned)((n * s.H + 3) / 4)), dim3(256), 0, st, (const double *)part, parts, dtable, n, s.H);
    return check_launch("hgq_relative_bias_bwd");
}

}  // namespace
}  // namespace hgq

using namespace hgq;

extern "C" int hgq_relative_bias_fwd(const void *scores, int64_t stride_b, int64_t stride_h, const float *table, void *out, int64_t B, int64_t H, int64_t T,
                                     int64_t S, const int *first, int m, int both, int64_t offset, const void *offsets, int offset_bytes, int type, void *stream) {
    int rc = check_bias("hgq_relative_bias_fwd", B, H, T, S, first, m, both, type, offset_bytes);
    if (rc || B == 0 || H == 0 || T == 0 || S == 0) return rc;
    if (!scores || !table || !out) return fail(HGQ_ERR_ARG, "hgq_relative_bias_fwd: null pointer");
    const BiasShape s = bias_shape(B, H, T, S, first, m, both, offset, offsets, offset_bytes, stride_b, stride_h);
    hipStream_t st = (hipStream_t)stream;
    return type == HGQ_TYPE_F32 ? add<float>(scores, table, out, s, st) : type == HGQ_TYPE_BF16 ? add<__bf16>(scores, table, out, s, st) : add<_Float16>(scores, table, out, s, st);
}

extern "C" int64_t hgq_relative_bias_bwd_workspace(int64_t B, int64_t H, int64_t T, int64_t S, int m, int both) {
    if (B < 0 || H < 0 || T < 0 || S < 0 || m < 2 || (both ? 2 : 1) * (int64_t)m > BIAS_BUCKETS) return -1;
    const int n = both ? 2 * m : m;
    return 2 * n * (512 * (256 / sums_threads(n)) + H);  // (the most parts there are, 8 bytes a bucket)
}

extern "C" int hgq_relative_bias_bwd(const void *dy, int64_t stride_b, int64_t stride_h, float *dtable, float *workspace, int64_t B, int64_t H, int64_t T, int64_t S,
                                     const int *first, int m, int both, int64_t offset, const void *offsets, int offset_bytes, int type, void *stream) {
    int rc = check_bias("hgq_relative_bias_bwd", B, H, T, S, first, m, both, type, offset_bytes);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (H == 0) return HGQ_OK;
    if (!dtable) return fail(HGQ_ERR_ARG, "hgq_relative_bias_bwd: null pointer");
    if (B == 0 || T == 0 || S == 0) return fill_f32(dtable, 0.0f, (both ? 2 : 1) * m * H, st);
    if (!dy || !workspace) return fail(HGQ_ERR_ARG, "hgq_relative_bias_bwd: null pointer");
    const BiasShape s = bias_shape(B, H, T, S, first, m, both, offset, offsets, offset_bytes, stride_b, stride_h);
    double *part = (double *)workspace;
    return type == HGQ_TYPE_F32 ? sums<float>(dy, dtable, part, s, st) : type == HGQ_TYPE_BF16 ? sums<__bf16>(dy, dtable, part, s, st) : sums<_Float16>(dy, dtable, part, s, st);
}
