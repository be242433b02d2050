// Loss of a student's logits z [rows, V] against a teacher's top logits t [rows, K] of the entries i [rows, K], temperature T:
//     q = softmax(z / T);   p_k = softmax(t / T) over the list, or exp(t_k / T - lse) with the teacher's own logarithm of its sum
//     loss_r = T^2 (sum_k p_k (log p_k - log q[i_k]) + p' log(p' / q'));   loss = sum_r w_r loss_r / rows
//     d loss / d z_j = w_r T / rows (P q_j - sum of p_k with i_k = j - p' q_j / q' outside the list),   P = sum p + p'
// p' = max(0, 1 - sum p) and q' are what lies outside the list (without the teacher's lse: p' = 0).
//
// With the lse the pass over a row leaves the list out, so that q' is a sum and no difference, with a maximum of its own, so that it does not vanish
// beside a list that holds nearly everything; the entries of the list are read again by themselves.  A bit per entry of the vocabulary, in LDS, says which
// are listed (one byte per access of eight entries).  Then every z_j of the pass has the gradient c a exp((z_j - m) / T) with two
// numbers m, a of its row, an entry of the list c (b exp((z_j - M) / T) - its p), c = w T / rows: the row's four numbers are what a backward call needs.
// Sums over a row are fp32 of at most 64 terms in a row and pairwise beyond, what is formed of the list's numbers is fp64.
#include "hgq_device.h"
#include "hgq_host.h"
#include "hgq_vector.h"

namespace hgq {

constexpr int DISTILL_LIST = 1024;           // entries of a list
constexpr int DISTILL_BITS = 1 << 18;        // entries whose bits a workgroup holds: 32 KB
constexpr int DISTILL_ENTRY = 16;            // bytes of LDS per entry of a list: p, index, logit

__host__ __device__ inline int bit_words(int entries) { return (entries + 63) / 64 * 2; }  // (p of the next row lies behind them)

struct DistillRows {
    const void *z, *t, *index;
    const float *lse, *weight, *upstream;
    float4 *stats;   // m, a, M, b
    double *losses;  // a workgroup's sum each
    float2 *parts;   // maximum and sum of each part of a row
    void *dz;
    int64_t rows, z_stride;
    double T, scale;  // scale: T^2 / rows
    float k_hi, k_lo;  // 1 / (T ln 2) in two pieces
    int V, K, t_type, wide_index, n_parts, grid_parts, part, leave_unit;
};

__device__ __forceinline__ float distill_logit(const DistillRows &a, int64_t at) {
    return a.t_type == HGQ_TYPE_F32    ? ((const float *)a.t)[at]
           : a.t_type == HGQ_TYPE_BF16 ? (float)((const __bf16 *)a.t)[at]
                                       : (float)((const _Float16 *)a.t)[at];
}

__device__ __forceinline__ int distill_index(const DistillRows &a, int64_t at) {
    const int64_t i = a.wide_index ? ((const int64_t *)a.index)[at] : ((const int32_t *)a.index)[at];
    return i >= 0 && i < a.V ? (int)i : -1;
}

// exp(d / T), d <= 0 or not a number.  fp32 outputs take the product d / (T ln 2) in two pieces (rounded once it is off by |d| 2^-24, which the
// exponential makes a relative error); 16-bit ones do not show it.
template <bool FINE>
__device__ __forceinline__ float exp_t(float d, float k_hi, float k_lo) {
    if (!FINE) return __builtin_amdgcn_exp2f(d * k_hi);
    const float hi0 = d * k_hi;
    const float hi = hi0 < -200.0f ? -200.0f : hi0;  // (the result is zero either way, infinities must not meet in the second piece)
    const float lo = hi0 < -200.0f ? 0.0f : fmaf(d, k_lo, fmaf(d, k_hi, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e, lo * HGQ_LN2, e);
}

// a maximum and the sum of exp((z - maximum) / T)
struct MaxSum {
    float m, s;
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

template <int TPR>
struct Team {  // the threads of one row
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;
    double *lds;  // WAVES numbers
    __device__ __forceinline__ void sync() const {
        if (TPR > 64) {
            __syncthreads();
        } else {  // one wavefront, its accesses in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
    }
    template <typename V>
    __device__ __forceinline__ V sum(V v) const {
        v = team_sum(v, TPR < 64 ? TPR : 64);
        if (TPR <= 64) return v;
        V *at = (V *)lds;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        v = team_sum(at[threadIdx.x & (WAVES - 1)], WAVES);
        __syncthreads();
        return v;
    }
    __device__ __forceinline__ float max(float v) const {
        v = team_max(v, TPR < 64 ? TPR : 64);
        if (TPR <= 64) return v;
        float *at = (float *)lds;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        v = team_max(at[threadIdx.x & (WAVES - 1)], WAVES);
        __syncthreads();
        return v;
    }
    __device__ __forceinline__ MaxSum join(MaxSum v, float k) const {
        const float m = max(v.m);
        return {m, sum(v.s * __builtin_amdgcn_exp2f((base_of(v.m) - base_of(m)) * k))};
    }
};

// z[at ...] with -inf behind `end` and, BITS, where an entry is listed (bits: of the entries from `lo` on)
template <typename T, bool BITS>
__device__ __forceinline__ Vec<T> distill_load(const T *z, int at, int end, const uint32_t *bits, int lo) {
    constexpr int N = Vec<T>::N;
    const T none = (T)-INFINITY;
    Vec<T> r;
    if (at + N <= end) {
        r = load_vec(z + at);
    } else {
        r = load_part(z + at, end - at, none);
    }
    if (BITS) {
        const uint32_t b = at < end ? bits[(at - lo) >> 5] >> ((at - lo) & 31) & ((1 << N) - 1) : 0;
        if (b) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (b >> e & 1) r.v[e] = none;
        }
    }
    return r;
}

template <typename T>
__device__ __forceinline__ float most_of(const Vec<T> &r) {
    float m = (float)r.v[0];
#pragma unroll
    for (int e = 1; e < Vec<T>::N; ++e) m = fmaxf(m, (float)r.v[e]);
    return m;
}

template <typename T>
__device__ __forceinline__ float exp_sum(const Vec<T> &r, float base, const DistillRows &a) {
    constexpr int N = Vec<T>::N;
    float e[N];
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = exp_t<sizeof(T) == 4>((float)r.v[k] - base, a.k_hi, a.k_lo);
#pragma unroll
    for (int w = N / 2; w; w /= 2)
#pragma unroll
        for (int k = 0; k < w; ++k) e[k] += e[k + w];
    return e[0];
}

// maximum and sum over z[lo, end) as the row is read once: the sum follows the maximum
template <typename T, int TPR, bool BITS>
__device__ __forceinline__ MaxSum distill_stream(const T *z, int lo, int end, const uint32_t *bits, int lane, const DistillRows &a) {
    constexpr int N = Vec<T>::N;
    MaxSum r = {-INFINITY, 0.0f};
    for (int at = lo + lane * N; at < end; at += TPR * N) {
        const Vec<T> v = distill_load<T, BITS>(z, at, end, bits, lo);
        const float m = most_of(v);
        if (m > r.m) r.s *= __builtin_amdgcn_exp2f((r.m - m) * a.k_hi), r.m = m;
        r.s += exp_sum(v, base_of(r.m), a);
    }
    return r;
}

template <typename T, int TPR>
__device__ __forceinline__ void distill_bits(uint32_t *bits, int lo, int end, const int *index, int K, int lane, const Team<TPR> &team) {
    for (int w = lane; w < (end - lo + 31) / 32; w += TPR) bits[w] = 0;
    team.sync();
    for (int k = lane; k < K; k += TPR) {
        const int i = index[k];
        if (i >= lo && i < end) atomicOr(&bits[(i - lo) >> 5], 1u << ((i - lo) & 31));
    }
    team.sync();
}

// Maximum and sum of part `blockIdx % n_parts` of a row.
template <typename T, bool REST>
__global__ __launch_bounds__(256) void distill_parts(const DistillRows a) {
    __shared__ double lds[4];
    extern __shared__ uint32_t distill_lds[];
    const Team<256> team = {lds};
    const int64_t row = blockIdx.x / a.n_parts;
    const int lo = (int)(blockIdx.x - row * a.n_parts) * a.part, end = min(a.V, lo + a.part), lane = threadIdx.x;
    int *index = (int *)distill_lds;
    uint32_t *bits = distill_lds + a.K;
    if (REST) {
        for (int k = lane; k < a.K; k += 256) index[k] = distill_index(a, row * a.K + k);
        team.sync();
        distill_bits<T>(bits, lo, end, index, a.K, lane, team);
    }
    const MaxSum r = team.join(distill_stream<T, 256, REST>((const T *)a.z + row * a.z_stride, lo, end, bits, lane, a), a.k_hi);
    if (lane == 0) a.parts[blockIdx.x] = make_float2(r.m, r.s);
}

// What the maximum and the sum of a row come from: the row itself, what distill_parts left, or a forward call's numbers
enum { FROM_ROW, FROM_PARTS, FROM_STATS };

// TPR threads take a row; HOLD elements of it stay in a thread's registers between the sum and the gradient (0: the row is read twice).
template <typename T, int TPR, bool REST, int FROM, int HOLD>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void distill_rows(const DistillRows a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR, N = Vec<T>::N, NV = HOLD ? HOLD / N : 1;
    constexpr bool FINE = sizeof(T) == 4;
    __shared__ double lds[THREADS / 64];
    extern __shared__ uint32_t distill_lds[];
    if (FROM == FROM_STATS && a.leave_unit && *a.upstream == 1.0f) return;  // dz holds this gradient

    const int slot = threadIdx.x / TPR, lane = threadIdx.x % TPR;
    const Team<TPR> team = {lds};
    const int64_t block = FROM == FROM_ROW ? blockIdx.x : blockIdx.x / a.grid_parts, row = block * ROWS + slot;
    const int lo = FROM == FROM_ROW ? 0 : (int)(blockIdx.x - block * a.grid_parts) * a.part, end = FROM == FROM_ROW ? a.V : min(a.V, lo + a.part);
    const int words = REST && FROM == FROM_ROW ? bit_words(a.V) : 0;
    double *p = (double *)((char *)distill_lds + slot * (DISTILL_ENTRY * a.K + 4 * words));  // (first the teacher's logits)
    int *index = (int *)(p + a.K);
    float *z_list = (float *)(index + a.K);
    uint32_t *bits = (uint32_t *)(z_list + a.K);

    double loss = 0;
    if (row < a.rows) {
        const T *z = (const T *)a.z + row * a.z_stride;
        T *dz = a.dz ? (T *)a.dz + row * a.V : nullptr;
        const double inv_T = 1.0 / a.T;
        const float weight = a.weight ? a.weight[row] : 1.0f;

        // the list
        float t_most = -INFINITY;
        for (int k = lane; k < a.K; k += TPR) {
            const int i = distill_index(a, row * a.K + k);
            const float t = i < 0 ? -INFINITY : distill_logit(a, row * a.K + k);
            index[k] = i, p[k] = t, z_list[k] = i < 0 ? -INFINITY : (float)z[i];
            if (t > t_most || t != t) t_most = t != t ? INFINITY : t;
        }
        t_most = team.max(t_most);
        team.sync();
        if (!(t_most > -INFINITY) || weight == 0.0f) {  // no entries, or no weight: no loss, no gradient
            if (dz)
                for (int at = lo + lane * N; at < end; at += TPR * N) {
                    Vec<T> zero;
#pragma unroll
                    for (int e = 0; e < N; ++e) zero.v[e] = (T)0.0f;
                    if (at + N <= end) store_vec(dz + at, zero);
                    else store_part(dz + at, zero, end - at);
                }
        } else {
            // maximum and sum of the row
            Vec<T> held[NV];
            MaxSum r = {-INFINITY, 0.0f};
            if (FROM == FROM_PARTS) {
                for (int c = lane; c < a.n_parts; c += TPR) {
                    const float2 q = a.parts[row * a.n_parts + c];
                    if (q.x > r.m) r.s *= __builtin_amdgcn_exp2f((r.m - q.x) * a.k_hi), r.m = q.x;
                    r.s += q.y * __builtin_amdgcn_exp2f((base_of(q.x) - base_of(r.m)) * a.k_hi);
                }
                r = team.join(r, a.k_hi);
            }
            if (FROM == FROM_ROW) {
                if (REST) distill_bits<T>(bits, 0, a.V, index, a.K, lane, team);
                if (HOLD) {
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) held[v] = distill_load<T, REST>(z, (v * TPR + lane) * N, a.V, bits, 0);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) r.m = fmaxf(r.m, most_of(held[v]));
                    r.m = team.max(r.m);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) r.s += exp_sum(held[v], base_of(r.m), a);
                    r.s = team.sum(r.s);
                } else {
                    r = team.join(distill_stream<T, TPR, REST>(z, 0, a.V, bits, lane, a), a.k_hi);
                }
            }

            // the teacher
            double log_sum = 0, p_sum = 0, p_rest = 0;
            if (REST) {
                log_sum = a.lse[row];
                for (int k = lane; k < a.K; k += TPR) p_sum += exp(p[k] * inv_T - log_sum);
                p_sum = team.sum(p_sum);
            } else {
                for (int k = lane; k < a.K; k += TPR) p_sum += exp_t<true>((float)p[k] - t_most, a.k_hi, a.k_lo);
                p_sum = team.sum(p_sum);
                log_sum = log(p_sum) + (double)t_most * inv_T;
            }

            // m, a of the pass and M, b of the list
            float m, pass, M, list;
            if (FROM == FROM_STATS) {
                const float4 s = a.stats[row];
                m = s.x, pass = s.y, M = s.z, list = s.w;
            } else {
                m = base_of(r.m);
                float most = r.m;
                double total = r.s;
                if (REST) {  // the whole row: with the list's entries, each once
                    for (int k = lane; k < a.K; k += TPR) most = fmaxf(most, z_list[k]);
                    most = team.max(most);
                    double s = 0;
                    for (int k = lane; k < a.K; k += TPR) {
                        const int i = index[k];
                        bool first = i >= 0;
                        for (int l = 0; l < k; ++l) first &= index[l] != i;
                        if (first) s += exp_t<true>(z_list[k] - most, a.k_hi, a.k_lo);
                    }
                    const double outside = r.s > 0.0f ? (double)r.s * exp(((double)r.m - most) * inv_T) : (double)r.s;
                    total = team.sum(s) + outside;
                    if (r.s > 0.0f) p_rest = fmax(0.0, 1.0 - p_sum);
                    if (lane == 0 && p_rest > 0) loss = p_rest * (log(p_rest) - (log((double)r.s) + ((double)r.m - most) * inv_T - log(total)));
                    pass = r.s == 0.0f ? 0.0f : (float)((p_sum + p_rest) * (outside / r.s) / total - p_rest / r.s);
                    list = (float)((p_sum + p_rest) / total);
                } else {
                    pass = list = (float)(1.0 / total);
                }
                M = base_of(most);
                const double log_total = log(total);
                for (int k = lane; k < a.K; k += TPR) {
                    const double log_p = p[k] * inv_T - log_sum, q = REST ? exp(log_p) : exp_t<true>((float)p[k] - t_most, a.k_hi, a.k_lo) / p_sum;
                    if (q != 0) loss += q * (log_p - (((double)z_list[k] - M) * inv_T - log_total));
                    p[k] = q;
                }
                loss = team.sum(loss) * weight * a.scale;
                if (a.stats && lane == 0 && lo == 0) a.stats[row] = make_float4(m, pass, M, list);
            }

            if (dz) {
                if (FROM == FROM_STATS)
                    for (int k = lane; k < a.K; k += TPR) p[k] = REST ? exp(p[k] * inv_T - log_sum) : exp_t<true>((float)p[k] - t_most, a.k_hi, a.k_lo) / p_sum;
                const float c = (float)(weight * a.scale * inv_T) * (FROM == FROM_STATS ? *a.upstream : 1.0f), ca = c * pass;
                if (HOLD) {
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        const int at = (v * TPR + lane) * N;
                        if (v * TPR * N >= a.V) continue;
                        Vec<T> o;
#pragma unroll
                        for (int e = 0; e < N; ++e) o.v[e] = (T)(ca * exp_t<FINE>((float)held[v].v[e] - m, a.k_hi, a.k_lo));
                        if (at + N <= a.V) store_vec(dz + at, o);
                        else if (at < a.V) store_part(dz + at, o, a.V - at);
                    }
                } else {
                    for (int at = lo + lane * N; at < end; at += TPR * N) {
                        const Vec<T> v = distill_load<T, false>(z, at, end, nullptr, 0);
                        Vec<T> o;
#pragma unroll
                        for (int e = 0; e < N; ++e) o.v[e] = (T)(ca * exp_t<FINE>((float)v.v[e] - m, a.k_hi, a.k_lo));
                        if (at + N <= end) store_vec(dz + at, o);
                        else store_part(dz + at, o, end - at);
                    }
                }
                // the list's entries, over what the pass wrote there
                __threadfence_block();
                team.sync();
                for (int k = lane; k < a.K; k += TPR) {
                    const int i = index[k];
                    if (i < lo || i >= end) continue;
                    double sum = 0;
                    for (int l = 0; l < a.K; ++l) sum += index[l] == i ? p[l] : 0.0;
                    dz[i] = (T)(c * (float)(list * (double)exp_t<true>(z_list[k] - M, a.k_hi, a.k_lo) - sum));
                }
            }
        }
    }
    if (FROM != FROM_STATS && lo == 0) {  // the workgroup's sum, its rows in order
        if (ROWS > 1) {
            __shared__ double sums[ROWS];
            __syncthreads();
            if (lane == 0) sums[slot] = loss;
            __syncthreads();
            if (threadIdx.x == 0) {
                loss = 0;
                for (int r = 0; r < ROWS; ++r) loss += sums[r];
            }
        }
        if (threadIdx.x == 0) a.losses[block] = loss;
    }
}

__global__ __launch_bounds__(1024) void distill_sum(const double *__restrict__ losses, int64_t n, float *__restrict__ loss) {
    __shared__ double lds[16];
    double s = 0;
    for (int64_t k = threadIdx.x; k < n; k += 1024) s += losses[k];
    const Team<1024> team = {lds};
    s = team.sum(s);
    if (threadIdx.x == 0) *loss = (float)s;
}

namespace {

constexpr int SPLIT_ROWS = 256;   // rows from which on a row has a workgroup to itself
constexpr int SPLIT_PART = 4096;  // entries of a part, at least

struct DistillPlan {
    int tpr, hold;        // threads per row, elements held
    int n_parts, part;    // of a row
    int64_t blocks;       // sums of losses
};

DistillPlan distill_plan(int64_t rows, int V, int K, bool rest) {
    DistillPlan p = {};
    p.tpr = V <= 64 && K <= 64 ? 8 : V <= 2048 && K <= 512 ? 64 : V <= 16384 ? 256 : 1024;
    p.hold = p.tpr == 8 ? 8 : p.tpr == 64 ? 32 : V <= 65536 ? 64 : 0;
    p.n_parts = 1, p.part = V;
    int64_t parts = 1;
    if (rows < SPLIT_ROWS && V >= 2 * SPLIT_PART) parts = (2 * SPLIT_ROWS + rows - 1) / rows;
    if (parts > V / SPLIT_PART) parts = V / SPLIT_PART;
    if (rest && parts < (V + DISTILL_BITS - 1) / DISTILL_BITS) parts = (V + DISTILL_BITS - 1) / DISTILL_BITS;
    if (parts > 1) {
        p.part = (int)(((V + parts - 1) / parts + 31) / 32 * 32);
        p.n_parts = (V + p.part - 1) / p.part;
        p.tpr = 256, p.hold = 0;
    }
    const int per = p.tpr < 256 ? 256 / p.tpr : 1;
    p.blocks = (rows + per - 1) / per;
    return p;
}

int check_distill(const char *what, int64_t rows, int64_t V, int64_t K, double T, int type, int t_type, int index_bytes) {
    if (rows < 0 || V < 1 || K < 1 || !(T > 0) || T > 3e38) return fail(HGQ_ERR_ARG, "%s: rows %lld, vocabulary %lld, list %lld, temperature %g", what, (long long)rows, (long long)V, (long long)K, T);
    if (type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16 || t_type < HGQ_TYPE_F32 || t_type > HGQ_TYPE_F16) return fail(HGQ_ERR_ARG, "%s: unknown type", what);
    if (index_bytes != 4 && index_bytes != 8) return fail(HGQ_ERR_ARG, "%s: indices of %d bytes", what, index_bytes);
    if (K > DISTILL_LIST) return fail(HGQ_ERR_UNSUPPORTED, "%s: a list of %lld entries, at most %d", what, (long long)K, DISTILL_LIST);
    if (V > 1 << 30 || rows > (int64_t)1 << 40) return fail(HGQ_ERR_UNSUPPORTED, "%s: %lld rows of %lld entries", what, (long long)rows, (long long)V);
    return HGQ_OK;
}

int64_t lds_of(const DistillRows &a, int tpr, bool bits, int entries) {
    return (int64_t)(tpr < 256 ? 256 / tpr : 1) * (DISTILL_ENTRY * a.K + (bits ? 4 * bit_words(entries) : 0));
}

template <typename T, int TPR, bool REST, int FROM, int HOLD>
int launch(const DistillRows &a, int64_t blocks, int64_t lds, hipStream_t st, const char *what) {
    constexpr int threads = TPR > 256 ? TPR : 256;
    if (blocks * threads > 0xffffffffLL) return fail(HGQ_ERR_UNSUPPORTED, "%s: too many rows", what);
    hipLaunchKernelGGL((distill_rows<T, TPR, REST, FROM, HOLD>), dim3((unsigned)blocks), dim3(threads), (size_t)lds, st, a);
    return check_launch(what);
}

template <typename T, bool REST>
int forward(DistillRows a, const DistillPlan &p, float *loss, hipStream_t st) {
    const char *what = "hgq_distill_topk_fwd";
    a.n_parts = p.n_parts, a.part = p.part;
    int rc;
    if (p.n_parts > 1) {
        const int64_t blocks = a.rows * p.n_parts;
        if (blocks * 256 > 0xffffffffLL) return fail(HGQ_ERR_UNSUPPORTED, "%s: too many rows", what);
        hipLaunchKernelGGL((distill_parts<T, REST>), dim3((unsigned)blocks), dim3(256), REST ? 4 * a.K + 4 * bit_words(p.part) : 0, st, a);
        if ((rc = check_launch(what))) return rc;
        a.grid_parts = a.dz ? p.n_parts : 1;  // (without a gradient one workgroup a row, which looks at the list alone)
        rc = launch<T, 256, REST, FROM_PARTS, 0>(a, a.rows * a.grid_parts, lds_of(a, 256, false, 0), st, what);
    } else {
        const int64_t lds = lds_of(a, p.tpr, REST, a.V);
        rc = p.tpr == 8     ? launch<T, 8, REST, FROM_ROW, 8>(a, p.blocks, lds, st, what)
             : p.tpr == 64  ? launch<T, 64, REST, FROM_ROW, 32>(a, p.blocks, lds, st, what)
             : p.tpr == 256 ? launch<T, 256, REST, FROM_ROW, 64>(a, p.blocks, lds, st, what)
             : p.hold       ? launch<T, 1024, REST, FROM_ROW, 64>(a, p.blocks, lds, st, what)
                            : launch<T, 1024, REST, FROM_ROW, 0>(a, p.blocks, lds, st, what);
    }
    if (rc) return rc;
    hipLaunchKernelGGL(distill_sum, dim3(1), dim3(1024), 0, st, (const double *)a.losses, p.blocks, loss);
    return check_launch(what);
}

template <typename T, bool REST>
int backward(DistillRows a, const DistillPlan &p, hipStream_t st) {
    const char *what = "hgq_distill_topk_bwd";
    a.grid_parts = p.n_parts, a.part = p.part;
    const int64_t lds = lds_of(a, p.tpr, false, 0), blocks = p.blocks * p.n_parts;
    return p.tpr == 8     ? launch<T, 8, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 64  ? launch<T, 64, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 256 ? launch<T, 256, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
                          : launch<T, 1024, REST, FROM_STATS, 0>(a, blocks, lds, st, what);
}

DistillRows arguments(const void *z, int64_t z_stride, const void *t, int t_type, const void *index, int index_bytes, const float *lse, const float *weight,
                      int64_t rows, int64_t V, int64_t K, double T) {
    DistillRows a = {};
    a.z = z, a.z_stride = z_stride, a.t = t, a.t_type = t_type, a.index = index, a.wide_index = index_bytes == 8, a.lse = lse, a.weight = weight;
    a.rows = rows, a.V = (int)V, a.K = (int)K, a.T = T, a.scale = T * T / (double)rows;
    const double k = 1.44269504088896340736 / T;
    a.k_hi = (float)k, a.k_lo = (float)(k - (double)a.k_hi);
    return a;
}

}  // namespace
}  // namespace hgq

using namespace hgq;

extern "C" int64_t hgq_distill_topk_workspace(int64_t rows, int64_t V, int64_t K, int rest) {
    if (check_distill("hgq_distill_topk_workspace", rows, V, K, 1.0, HGQ_TYPE_F32, HGQ_TYPE_F32, 4)) return -1;
    const DistillPlan p = distill_plan(rows, (int)V, (int)K, rest);
    return 2 * p.blocks + (p.n_parts > 1 ? 2 * rows * p.n_parts : 0);
}

extern "C" int hgq_distill_topk_fwd(const void *z, int64_t z_stride, const void *t, int t_type, const void *index, int index_bytes, const float *lse,
                                    const float *weight, float *loss, float *stats, void *dz, float *workspace, int64_t rows, int64_t V, int64_t K,
                                    double T, int type, void *stream) {
    const char *what = "hgq_distill_topk_fwd";
    int rc = check_distill(what, rows, V, K, T, type, t_type, index_bytes);
    if (rc) return rc;
    if (!loss) return fail(HGQ_ERR_ARG, "%s: null pointer", what);
    if (rows == 0) return fill_f32(loss, 0.0f, 1, (hipStream_t)stream);
    if (!z || !t || !index || !workspace) return fail(HGQ_ERR_ARG, "%s: null pointer", what);
    if (z_stride < 0) return fail(HGQ_ERR_ARG, "%s: rows of logits must not run backwards", what);
    DistillRows a = arguments(z, z_stride, t, t_type, index, index_bytes, lse, weight, rows, V, K, T);
    const DistillPlan p = distill_plan(rows, (int)V, (int)K, lse != nullptr);
    a.stats = (float4 *)stats, a.dz = dz, a.losses = (double *)workspace, a.parts = (float2 *)(workspace + 2 * p.blocks);
    hipStream_t st = (hipStream_t)stream;
    if (lse) return type == HGQ_TYPE_F32 ? forward<float, true>(a, p, loss, st) : type == HGQ_TYPE_BF16 ? forward<__bf16, true>(a, p, loss, st) : forward<_Float16, true>(a, p, loss, st);
    return type == HGQ_TYPE_F32 ? forward<float, false>(a, p, loss, st) : type == HGQ_TYPE_BF16 ? forward<__bf16, false>(a, p, loss, st) : forward<_Float16, false>(a, p, loss, st);
}

extern "C" int hgq_distill_topk_bwd(const void *z, int64_t z_stride, const void *t, int t_type, const void *index, int index_bytes, const float *lse,
                                    const float *weight, const float *upstream, const float *stats, void *dz, int holds_unit, int64_t rows, int64_t V,
                                    int64_t K, double T, int type, void *stream) {
    const char *what = "hgq_distill_topk_bwd";
    int rc = check_distill(what, rows, V, K, T, type, t_type, index_bytes);
    if (rc) return rc;
    if (rows == 0) return HGQ_OK;
    if (!z || !t || !index || !upstream || !stats || !dz) return fail(HGQ_ERR_ARG, "%s: null pointer", what);
    if (z_stride < 0) return fail(HGQ_ERR_ARG, "%s: rows of logits must not run backwards", what);
    DistillRows a = arguments(z, z_stride, t, t_type, index, index_bytes, lse, weight, rows, V, K, T);
    a.stats = (float4 *)stats, a.dz = dz, a.upstream = upstream, a.leave_unit = holds_unit;
    const DistillPlan p = distill_plan(rows, (int)V, (int)K, lse != nullptr);
    hipStream_t st = (hipStream_t)stream;
    if (lse) return type == HGQ_TYPE_F32 ? backward<float, true>(a, p, st) : type == HGQ_TYPE_BF16 ? backward<__bf16, true>(a, p, st) : backward<_Float16, true>(a, p, st);
    return type == HGQ_TYPE_F32 ? backward<float, false>(a, p, st) : type == HGQ_TYPE_BF16 ? backward<__bf16, false>(a, p, st) : backward<_Float16, false>(a, p, st);
}
