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
constexpr int ADD_WGS = 2048;
constexpr int BIAS_NEAR = 4096;  // distances whose bucket a workgroup looks up; beyond, where buckets still change there, it searches

struct BiasShape {
    int first[BIAS_BUCKETS];  // of buckets 1 .. m - 1
    int64_t stride_b, stride_h, offset;
    const void *offsets;  // [B] (int32 or int64) or null
    int B, H, S, TS, m, both, wide, near, chunk, chunks, tiles, align, per, groups;  // per: threads for a plane, groups: planes (of other sequences) side by side where it takes few
    uint32_t magic, shift;  // of the division by S
    __device__ __forceinline__ int row_of(int e) const { return (int)((__umulhi((uint32_t)e, magic) + (uint32_t)e) >> shift); }
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

// Offsets beyond all distances that there are (queries and keys: below 2^28, first distances: up to 2^30) are as good as the first such one.
__device__ __forceinline__ int offset_of(const BiasShape &s, int b) {
    const int64_t o = !s.offsets ? s.offset : s.wide ? ((const int64_t *)s.offsets)[b] : (int64_t)((const int32_t *)s.offsets)[b];
    constexpr int64_t far = ((int64_t)1 << 30) + (1 << 28);
    return (int)(o < -far ? -far : o > far ? far : o);
}

// By how many elements a plane's accesses begin early, so that a wavefront's lie in lines of its own (8 x 16 x 2047 x 2047 bfloat16: forward 513 -> 462 us, the table's
// gradient 265 -> 222 us); s.align: elements of a line, 1 where planes lie there already, or differently in the sequences of a run.
template <typename T>
__device__ __forceinline__ int shift_of(const BiasShape &s, const T *plane) {
    return (int)((uintptr_t)plane / sizeof(T) & (uintptr_t)(s.align - 1));
}

// A workgroup takes tiles t, t + stride, ... of a head's plane (256 accesses each) and a run of the batch.
template <typename T, int AHEAD, bool THROUGH, bool TINY>
__global__ __launch_bounds__(256) void relative_bias_add(const T *__restrict__ scores, const float *__restrict__ table, T *__restrict__ out, int stride, const BiasShape s) {
    constexpr int N = Vec<T>::N;
    extern __shared__ float by_distance[];  // [2 near + 1], then the first distances
    int *first = (int *)(by_distance + 2 * s.near + 1);
    for (int k = threadIdx.x; k < s.m - 1; k += 256) first[k] = s.first[k];
    __syncthreads();
    int block = blockIdx.x;
    const int tile0 = block % stride;
    block /= stride;
    const int h = block % s.H, b0 = block / s.H * s.chunk, b1 = min(s.B, b0 + s.chunk);
    for (int k = threadIdx.x; k <= 2 * s.near; k += 256) by_distance[k] = table[bucket_of(s, first, k - s.near) * s.H + h];
    __syncthreads();
    const bool beyond = s.first[s.m - 2] > s.near;
    const int64_t step = (int64_t)s.H * s.TS;
    const int group = threadIdx.x / s.per, thread = threadIdx.x - group * s.per;
    const int shift = TINY ? 0 : shift_of(s, out + ((int64_t)b0 * s.H + h) * s.TS);
    for (int tile = tile0; tile < s.tiles; tile += stride) {
        const int at = (tile * 256 + thread) * N - shift;
        if (at >= s.TS || group >= s.groups) return;
        if (at + N <= 0) continue;
        const int e0 = TINY ? 0 : max(0, min(at, s.TS - N)), i0 = s.row_of(e0), j0 = e0 - i0 * s.S;
        float bias[N];
        const int first_b = b0 + group;
        for (int b = first_b; b < b1; b += AHEAD * s.groups) {
            const T *from = scores + b * s.stride_b + h * s.stride_h + e0;
            T *to = out + ((int64_t)b * s.H + h) * s.TS + e0;
            Vec<T> v[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const T *p = from + min(a * s.groups, b1 - 1 - b) * s.stride_b;
                if (TINY) v[a] = load_part(p, s.TS, (T)0.0f);
                else v[a] = load_vec<T, THROUGH>(p);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (b + a * s.groups >= b1) break;
                if ((a == 0 && b == first_b) || s.offsets) {
                    const int offset = offset_of(s, b + a * s.groups);
                    int i = i0, j = j0;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int d = j - i - offset;
                        bias[e] = by_distance[max(-s.near, min(s.near, d)) + s.near];
                        if (++j == s.S) j = 0, ++i;
                    }
                    if (beyond) {
                        i = i0, j = j0;
                        for (int e = 0; e < N; ++e) {
                            const int d = j - i - offset;
                            if (abs(d) > s.near) bias[e] = table[bucket_of(s, first, d) * s.H + h];
                            if (++j == s.S) j = 0, ++i;
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < N; ++e) v[a].v[e] = (T)((float)v[a].v[e] + bias[e]);
                // (the first and the last access write some of what their neighbour writes, once more)
                if (TINY) store_part(to + a * s.groups * step, v[a], s.TS);
                else store_vec<T, THROUGH>(to + a * s.groups * step, v[a]);
            }
        }
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

// Workgroup w of a head takes items w, w + parts, ... - an item: TILES tiles of the plane and a run of the batch, which is read SEQS sequences at a time (with
// more than one tile a run has no more than that).  While one such round is added up, the next one's loads are on their way.  parts [H][parts][n].
// The last access of a plane ends with it, and its first elements are the one before's again: no access is cut (a load that may be either whole or cut is
// taken apart into elements where it arrives, and waited for there: 357 us instead of 205 at 8 x 16 x 2048 x 2048 bfloat16).  TINY: planes of less than one access.
template <typename T, int SEQS, int TILES, bool TINY>
__global__ __launch_bounds__(256) void relative_bias_sums(const T *__restrict__ dy, double *__restrict__ part, int parts, const BiasShape s) {
    constexpr int N = Vec<T>::N, LOADS = SEQS * TILES;
    extern __shared__ double bias_lds[];
    const int n_buckets = s.both ? 2 * s.m : s.m, threads = blockDim.x;
    int *first = (int *)(bias_lds + n_buckets * threads);
    uint8_t *near = (uint8_t *)(first + BIAS_BUCKETS);
    const bool beyond = s.first[s.m - 2] > s.near;
    const int h = blockIdx.x / parts, w = blockIdx.x - h * parts;
    BiasRun run = {bias_lds, threads, -1, 0.0};
    const int sets = (s.tiles + TILES - 1) / TILES, rounds = TILES > 1 ? 1 : (s.chunk + SEQS * s.groups - 1) / (SEQS * s.groups);
    const int group = threadIdx.x / s.per, thread = threadIdx.x - group * s.per;
    const int64_t items = (int64_t)sets * s.chunks;
    double sum[N] = {};

    struct Step {
        int64_t item;
        int c, tile, round, shift, offset;  // (with offsets of their own, runs are of one sequence)
    };
    auto step_of = [&](int64_t item) {
        const int c = min((int)(item / sets), s.chunks - 1);
        return Step{item, c, (int)min(item - (int64_t)c * sets, (int64_t)sets) * TILES, 0, TINY ? 0 : shift_of(s, dy + (int64_t)c * s.chunk * s.stride_b + h * s.stride_h), offset_of(s, c * s.chunk)};
    };
    auto after = [&](const Step &k) { return k.round + 1 < rounds ? Step{k.item, k.c, k.tile, k.round + 1, k.shift, k.offset} : step_of(k.item + parts); };
    // (32 bits hold it: a plane has at most 2^31 - 2^16 elements, and the tiles behind it end less than 2^15 later)
    auto first_of = [&](const Step &k, int t) { return group >= s.groups ? s.TS : ((k.tile + t) * threads + thread) * N - k.shift; };

    auto ask = [&](const Step &k, Vec<T> *v) {  // beyond the run and the last item: what is there already, once more
        const int b1 = min(s.B, (k.c + 1) * s.chunk), b = min(b1 - 1, k.c * s.chunk + k.round * SEQS * s.groups + group);
        const T *plane = dy + b * s.stride_b + h * s.stride_h;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const T *from = plane + max(0, min(first_of(k, t), s.TS - N));
#pragma unroll
            for (int a = 0; a < SEQS; ++a) {
                const T *at = from + min(a * s.groups, b1 - 1 - b) * s.stride_b;
                if (TINY) v[t * SEQS + a] = load_part(at, s.TS, (T)0.0f);
                else v[t * SEQS + a] = load_vec(at);
            }
        }
    };

    auto bucket = [&](int d) {
        int k = near[max(-s.near, min(s.near, d)) + s.near];
        if (beyond && abs(d) > s.near) k = bucket_of(s, first, d);
        return k;
    };

    auto take = [&](const Step &k, const Vec<T> *v) {
        const int left = min(s.B, (k.c + 1) * s.chunk) - (k.c * s.chunk + k.round * SEQS * s.groups + group);  // sequences from this thread's first one on
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float g[SEQS];
#pragma unroll
                for (int a = 0; a < SEQS; ++a) g[a] = SEQS == 1 || a * s.groups < left ? (float)v[t * SEQS + a].v[e] : 0.0f;
#pragma unroll
                for (int d = SEQS / 2; d; d /= 2)
#pragma unroll
                    for (int a = 0; a < d; ++a) g[a] += g[a + d];
                f[e] = g[0];
                if (TILES == 1) sum[e] += g[0];
            }
            if (k.round + 1 < rounds) continue;
            const int at = first_of(k, t);
            if (at < s.TS && at > -N && (SEQS > 1 || left > 0)) {
                // elements skip .. n - 1 are this access' own
                const int e0 = TINY ? 0 : max(0, min(at, s.TS - N)), skip = max(0, at - e0), n = TINY ? s.TS : N + min(0, at - e0), i0 = s.row_of(e0), j0 = e0 - i0 * s.S;
                const int d0 = j0 - i0 - k.offset, k0 = bucket(d0), k1 = bucket(d0 + N - 1);
                if (!TINY && j0 + N <= s.S && k0 == k1) {
                    double all[N];
                    constexpr int FOLDED = TILES == 1 ? N : N * SEQS / 8 > 1 ? N * SEQS / 8 : 1;  // sums of up to eight terms
                    if (skip > 0 || n < N) {  // (a plane's first or last access)
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (e < skip || e >= n) f[e] = 0.0f, sum[e] = 0.0;
                    }
                    if (TILES > 1) {
#pragma unroll
                        for (int d = N / 2; d >= FOLDED; d /= 2)
#pragma unroll
                            for (int e = 0; e < d; ++e) f[e] += f[e + d];
                    }
#pragma unroll
                    for (int e = 0; e < FOLDED; ++e) all[e] = TILES > 1 ? (double)f[e] : sum[e];
#pragma unroll
                    for (int d = FOLDED / 2; d; d /= 2)
#pragma unroll
                        for (int e = 0; e < d; ++e) all[e] += all[e + d];
                    run.add(k0, all[0]);
                } else {
                    int d = d0, j = j0, of[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        of[e] = bucket(d++);
                        if (++j == s.S) j = 0, d -= s.S + 1;  // the next query's first key
                    }
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (e >= skip && e < n) run.add(of[e], TILES > 1 ? (double)f[e] : sum[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0;
        }
    };

    Vec<T> even[LOADS], odd[LOADS];
    Step k = step_of(w);
    ask(k, even);  // and the tables meanwhile
    for (int e = threadIdx.x; e < s.m - 1; e += threads) first[e] = s.first[e];
    for (int e = threadIdx.x; e < n_buckets * threads; e += threads) bias_lds[e] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e <= 2 * s.near; e += threads) near[e] = (uint8_t)bucket_of(s, first, e - s.near);
    __syncthreads();
    while (k.item < items) {
        const Step k1 = after(k);
        ask(k1, odd);
        take(k, even);
        if (k1.item >= items) break;
        k = after(k1);
        ask(k, even);
        take(k1, odd);
    }
    run.flush();
    __syncthreads();
    // a team of lanes for each bucket; neighbouring teams begin at neighbouring bins, which lie in other banks
    const int team = min(64, max(1, threads / (1 << (32 - __clz(n_buckets - 1))))), lane = threadIdx.x & (team - 1);
    for (int k = threadIdx.x / team; k < n_buckets; k += threads / team) {
        double v = 0;
        for (int t = lane; t < threads; t += team) v += bias_lds[k * threads + ((t + k * team) & (threads - 1))];
        v = team_sum(v, team);
        if (lane == 0) part[(int64_t)blockIdx.x * n_buckets + k] = v;
    }
}

// dtable [n, H] from [H][parts][n], elements `from` on: a wavefront for each
__global__ __launch_bounds__(256) void relative_bias_join(const double *__restrict__ part, int parts, float *__restrict__ dtable, int n, int H, int from) {
    const int at = from + blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
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
    if (B > 1 << 30 || H > 1 << 20 || T >= 1 << 28 || S >= 1 << 28 || T * S > INT32_MAX - (1 << 16)) return fail(HGQ_ERR_UNSUPPORTED, "%s: %lld x %lld positions", what, (long long)T, (long long)S);
    return HGQ_OK;
}

BiasShape bias_shape(int64_t B, int64_t H, int64_t T, int64_t S, const int *first, int m, int both, int64_t offset, const void *offsets, int offset_bytes,
                     int64_t stride_b, int64_t stride_h) {
    BiasShape s = {};
    for (int k = 0; k + 1 < m; ++k) s.first[k] = first[k];
    s.B = (int)B, s.H = (int)H, s.S = (int)S, s.TS = (int)(T * S), s.m = m, s.both = both, s.offset = offset, s.offsets = offsets, s.wide = offset_bytes == 8;
    s.stride_b = stride_b, s.stride_h = stride_h;
    // the distances whose bucket is looked up: no more than there are
    int64_t reach = BIAS_NEAR;
    if (!offsets && offset > -reach && offset < reach) {
        const int64_t ahead = S - 1 - offset, behind = T - 1 + offset, most = ahead > behind ? ahead : behind;
        reach = most < 1 ? 1 : most < reach ? most : reach;
    }
    s.near = (int)(first[m - 2] < reach ? first[m - 2] : reach);
    // e / S = (hi(e magic) + e) >> shift for e < 2^31, with magic = floor(2^32 (2^shift - S) / S) + 1 and 2^shift the first power of two that is not below S
    while (((int64_t)1 << s.shift) < S) ++s.shift;
    s.magic = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s.shift) - (uint64_t)S)) / (uint64_t)S + 1);
    return s;
}

// Tiles of the plane, and runs of the batch for `wanted` workgroups; planes lie at `base`, stride_b and stride_h elements apart.  each: a run's sequences may lie differently
// (and have offsets of their own).
template <typename T>
void cut(BiasShape &s, int64_t threads, int64_t wanted, const void *base, int64_t stride_b, int64_t stride_h, bool each) {
    constexpr int N = Vec<T>::N, LINE = 128 / sizeof(T);
    const int64_t per = threads * N, tiles = (s.TS + per - 1) / per;
    s.per = s.TS <= threads / 2 * N ? (s.TS + N - 1) / N : (int)threads, s.groups = (int)threads / s.per;
    const int64_t most = ((int64_t)s.B + s.groups - 1) / s.groups;
    int64_t chunks = (wanted + tiles * s.H - 1) / (tiles * s.H);
    if (chunks > most) chunks = most;
    if (s.offsets && !each) chunks = s.B;
    if (each && stride_b % LINE != 0 && s.TS >= 1 << 16) chunks = s.B;
    s.chunk = (int)((s.B + chunks - 1) / chunks);
    s.chunks = (s.B + s.chunk - 1) / s.chunk;
    const bool there = (uintptr_t)base % 128 == 0 && (s.B == 1 || stride_b % LINE == 0) && (s.H == 1 || stride_h % LINE == 0);
    s.align = there || s.groups > 1 || s.TS < 2 * LINE ? 1 : LINE;
    while (s.chunk > 1 && s.align > 1 && stride_b % s.align != 0) s.align /= 2;
    if (s.align < N) s.align = 1;
    s.tiles = (int)((s.TS + s.align - 1 + per - 1) / per);
}

int sums_threads(int n) { return n <= 16 ? 256 : n <= 32 ? 128 : 64; }  // 32 KB of bins with 16, 32 and 64 buckets: four workgroups a compute unit, three beside the longest table of distances

int sums_parts(const BiasShape &s, int threads, int tiles) {
    const int64_t items = (int64_t)((s.tiles + tiles - 1) / tiles) * s.chunks;
    int64_t parts = (512 * (256 / threads) + s.H - 1) / s.H;
    return (int)(items < parts ? items : parts);
}

template <typename T>
auto add_kernel(const BiasShape &s, bool through) {
    if (s.TS < Vec<T>::N) return relative_bias_add<T, 4, false, true>;
    if ((s.chunk + s.groups - 1) / s.groups < 4) return through ? relative_bias_add<T, 1, true, false> : relative_bias_add<T, 1, false, false>;
    return through ? relative_bias_add<T, 4, true, false> : relative_bias_add<T, 4, false, false>;
}

template <typename T>
int add(const void *scores, const float *table, void *out, BiasShape s, hipStream_t st) {
    cut<T>(s, 256, 2048, out, (int64_t)s.H * s.TS, s.TS, true);
    // a workgroup's table of biases takes it some 2 us: tiles in turn
    int64_t stride = ADD_WGS / ((int64_t)s.H * s.chunks) + 1;
    if (stride > s.tiles) stride = s.tiles;
    const int64_t blocks = stride * s.H * s.chunks;
    if (blocks * 256 > 0xffffffffLL) return fail(HGQ_ERR_UNSUPPORTED, "hgq_relative_bias_fwd: too many scores");
    const bool through = (int64_t)s.B * s.H * s.TS * (int64_t)sizeof(T) * 2 > (int64_t)256 << 20;
    hipLaunchKernelGGL(add_kernel<T>(s, through), dim3((unsigned)blocks), dim3(256), 4 * (2 * s.near + 1 + BIAS_BUCKETS), st, (const T *)scores, table, (T *)out,
                       (int)stride, s);
    return check_launch("hgq_relative_bias_fwd");
}

template <typename T, int SEQS, int TILES, bool TINY>
int sums_of(const void *dy, double *part, int parts, int threads, const BiasShape &s, hipStream_t st) {
    const int n = s.both ? 2 * s.m : s.m, lds = 8 * n * threads + 4 * BIAS_BUCKETS + 2 * s.near + 1;
    // (more than 112 buckets; per device, so it is asked for at every such call)
    if (lds > 64 << 10 && hipFuncSetAttribute((const void *)relative_bias_sums<T, SEQS, TILES, TINY>, hipFuncAttributeMaxDynamicSharedMemorySize, 80 << 10) != hipSuccess) {
        (void)hipGetLastError();
        return fail(HGQ_ERR_LAUNCH, "hgq_relative_bias_bwd: cannot reserve LDS");
    }
    hipLaunchKernelGGL((relative_bias_sums<T, SEQS, TILES, TINY>), dim3((unsigned)(parts * s.H)), dim3(threads), lds, st, (const T *)dy, part, parts, s);
    return check_launch("hgq_relative_bias_bwd");
}

template <typename T>
int sums(const void *dy, float *dtable, double *part, BiasShape s, hipStream_t st) {
    const int n = s.both ? 2 * s.m : s.m, threads = sums_threads(n);
    // a workgroup's bins and tables take it some 5 us: 16 KB of terms at least
    const int64_t terms = (int64_t)s.B * s.H * s.TS * sizeof(T) >> 14;
    cut<T>(s, threads, terms < 1 ? 1 : terms < 1024 ? terms : 1024, dy, s.stride_b, s.stride_h, false);
    const int each = s.offsets ? 1 : (s.chunk + s.groups - 1) / s.groups, seqs = each >= 5 ? 8 : each >= 3 ? 4 : each, parts = sums_parts(s, threads, 8 / seqs);
    const bool tiny = s.TS < Vec<T>::N;
    int rc = (tiny        ? seqs == 8 ? sums_of<T, 8, 1, true> : seqs == 4 ? sums_of<T, 4, 2, true> : seqs == 2 ? sums_of<T, 2, 4, true> : sums_of<T, 1, 8, true>
              : seqs == 8 ? sums_of<T, 8, 1, false>
              : seqs == 4 ? sums_of<T, 4, 2, false>
              : seqs == 2 ? sums_of<T, 2, 4, false>
                          : sums_of<T, 1, 8, false>)(dy, part, parts, threads, s, st);
    if (rc) return rc;
    constexpr int most = 1 << 25;  // elements of a launch (one of 2^32 threads or more runs some of them, and says nothing)
    for (int from = 0; from < n * s.H && !rc; from += most) {
        const int left = n * s.H - from, here = left < most ? left : most;
        hipLaunchKernelGGL(relative_bias_join, dim3((unsigned)((here + 3) / 4)), dim3(256), 0, st, (const double *)part, parts, dtable, n, s.H, from);
        rc = check_launch("hgq_relative_bias_bwd");
    }
    return rc;
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
