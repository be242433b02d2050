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
#include <algorithm>

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
    float *loss;     // where there is one workgroup
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

// exp(x) and log(x) of numbers in 64 bits with an error of fp32's rounding: what is large of them - whole powers of two - stays in 64 bits.  (The
// library's take some hundred instructions in 64 bits, for each row more than the row's own where the vocabulary is small.  The teacher's lse is a number in fp32, whose own
// half step moves p by as much.)
__device__ __forceinline__ double exp_64(double x) {
    const double two = x * 1.4426950408889634074, whole = __builtin_rint(two);
    if (!(two > -1000.0)) return two != two ? two : 0.0;
    return ldexp((double)__builtin_amdgcn_exp2f((float)(two - whole)), (int)fmin(whole, 1100.0));
}

__device__ __forceinline__ double log_64(double x) {
    int e;
    const float f = (float)frexp(x, &e);  // [0.5, 1)
    return x > 0.0 && x < INFINITY ? (double)e * 0.69314718055994530942 + (double)(__builtin_amdgcn_logf(f) * 0.69314718f) : x == 0.0 ? (double)-INFINITY : x < 0.0 ? (double)__builtin_nanf("") : x;
}

// a maximum and the sum of exp((z - maximum) / T)
struct MaxSum {
    float m, s;
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// What is added up over a row: the pass, the list's entries (each once), and the teacher's p and p (log p - z / T).
struct RowSums {
    MaxSum pass, list;
    double p, a;
};

// (a side without entries has the maximum -inf, its factor is exp(-inf) = 0: with a number in place of its -inf the factor overflows beside a low maximum, and
// zero times that is not a number)
__device__ __forceinline__ float down_to(float m, float most, float k) { return __builtin_amdgcn_exp2f((m - base_of(most)) * k); }

__device__ __forceinline__ MaxSum team_join(MaxSum v, int width, float k) {
    const float m = team_max(v.m, width);
    return {m, team_sum(v.s * down_to(v.m, m, k), width)};
}

__device__ __forceinline__ RowSums team_join(const RowSums &v, int width, float k) {
    return {team_join(v.pass, width, k), team_join(v.list, width, k), team_sum(v.p, width), team_sum(v.a, width)};
}

template <int TPR>
struct Team {  // the threads of one row
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;
    RowSums *lds;  // one for each wavefront
    __device__ __forceinline__ void sync() const {
        if (TPR > 64) {
            __syncthreads();
        } else {  // one wavefront, its accesses in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
    }
    __device__ __forceinline__ float max(float v) const {
        v = team_max(v, TPR < 64 ? TPR : 64);
        if (TPR <= 64) return v;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6].pass.m = v;
        __syncthreads();
        return team_max(lds[threadIdx.x & (WAVES - 1)].pass.m, WAVES);
    }
    template <typename V>
    __device__ __forceinline__ V join(V v, float k) const {
        v = team_join(v, TPR < 64 ? TPR : 64, k);
        if (TPR <= 64) return v;
        __syncthreads();  // (max's)
        V *at = (V *)lds;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        return team_join(at[threadIdx.x & (WAVES - 1)], WAVES, k);
    }
};

// One access of a row: elements `own` .. of z[at ...] are its own, the first ones may be another thread's once more - a row's last access ends with the row, so
// that no access is cut (one that may be whole or cut is taken apart where it arrives, and waited for there).  Rows that are shorter than an access
// (teams of eight) are filled with -inf.
template <typename T, int TPR>
struct Piece {
    static constexpr int N = Vec<T>::N;
    int at, own;
    __device__ __forceinline__ Piece(int wanted, int end) {
        at = TPR > 8 ? min(wanted, end - N) : wanted;
        own = min(N, wanted - at);
    }
    __device__ __forceinline__ Vec<T> load(const T *z, int end) const {
        if (TPR > 8) return load_vec(z + at);
        return at + N <= end ? load_vec(z + at) : load_part(z + at, end - at, (T)-INFINITY);
    }
    // -inf where an entry is listed (bits: of the entries from `lo` on) or another thread's, whose list this one does not look at
    __device__ __forceinline__ void leave_listed(Vec<T> &r, const uint32_t *bits, int lo, int end) const {
        if (at >= end) return;
        const int first = at - lo;
        uint32_t b;
        if (own == 0) {
            b = bits[first >> 5] >> (first & 31) & ((1 << N) - 1);
        } else {
            b = (1 << own) - 1;
            for (int e = own; e < N; ++e) b |= (bits[(first + e) >> 5] >> ((first + e) & 31) & 1) << e;
        }
        if (b) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (b >> e & 1) r.v[e] = (T)-INFINITY;
        }
    }
    template <bool THROUGH>
    __device__ __forceinline__ void store(T *z, const Vec<T> &r, int end) const {
        if (own == 0 && at + N <= end) {
            store_vec<T, THROUGH>(z + at, r);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e >= own && at + e < end) z[at + e] = r.v[e];
        }
    }
};

template <typename T>
__device__ __forceinline__ float most_of(const Vec<T> &r) {
    float m = (float)r.v[0];
#pragma unroll
    for (int e = 1; e < Vec<T>::N; ++e) m = fmaxf(m, (float)r.v[e]);
    return m;
}

template <typename T>
__device__ __forceinline__ float exp_sum(const Vec<T> &r, int own, float base, const DistillRows &a) {
    constexpr int N = Vec<T>::N;
    float e[N];
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = exp_t<sizeof(T) == 4>((float)r.v[k] - base, a.k_hi, a.k_lo);
    if (own) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < own) e[k] = 0.0f;
    }
#pragma unroll
    for (int w = N / 2; w; w /= 2)
#pragma unroll
        for (int k = 0; k < w; ++k) e[k] += e[k + w];
    return e[0];
}

constexpr int AHEAD = 4;  // accesses of a thread in flight

// maximum and sum over z[lo, end) as the row is read once: the sum follows the maximum
template <typename T, int TPR, bool BITS>
__device__ __forceinline__ MaxSum distill_stream(const T *z, int lo, int end, const uint32_t *bits, int lane, const DistillRows &a) {
    constexpr int N = Vec<T>::N;
    MaxSum r = {-INFINITY, 0.0f};
    for (int at = lo + lane * N; at < end; at += AHEAD * TPR * N) {
        Vec<T> v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = Piece<T, TPR>(at + k * TPR * N, end).load(z, end);
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (BITS) Piece<T, TPR>(at + k * TPR * N, end).leave_listed(v[k], bits, lo, end);
            m = fmaxf(m, most_of(v[k]));
        }
        if (m > r.m) r.s *= __builtin_amdgcn_exp2f((r.m - m) * a.k_hi), r.m = m;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const Piece<T, TPR> p(at + k * TPR * N, end);
            if (p.own < N) r.s += exp_sum(v[k], p.own, base_of(r.m), a);
        }
    }
    return r;
}

// the listed entries' bits; *again is set where an index comes twice
template <typename T, int TPR>
__device__ __forceinline__ void distill_bits(uint32_t *bits, int lo, int end, const int *index, int K, int lane, const Team<TPR> &team, int *again) {
    for (int w = lane; w < (end - lo + 31) / 32; w += TPR) bits[w] = 0;
    team.sync();
    for (int k = lane; k < K; k += TPR) {
        const int i = index[k];
        if (i >= lo && i < end) {
            const uint32_t bit = 1u << ((i - lo) & 31);
            if (atomicOr(&bits[(i - lo) >> 5], bit) & bit) *again = 1;
        }
    }
    team.sync();
}

// Without those bits: indices into a table of at least twice as many places, each at the first free one from its own on.  (Comparing all with all took nine tenths
// of the time of 25299 rows of 816 entries with lists of 178.)
__host__ __device__ inline int table_places(int K) {
    int n = 8;
    while (n < 2 * K) n *= 2;
    return n;
}

template <int TPR>
__device__ __forceinline__ void find_again(int *table, const int *index, int K, int lane, const Team<TPR> &team, int *again) {
    const int places = table_places(K);
    for (int k = lane; k < places; k += TPR) table[k] = -1;
    team.sync();
    for (int k = lane; k < K; k += TPR) {
        const int i = index[k];
        if (i < 0) continue;
        for (int at = (uint32_t)i * 2654435761u >> 8 & (places - 1);; at = (at + 1) & (places - 1)) {  // (half of the places stay free)
            const int there = atomicCAS(&table[at], -1, i);
            if (there == -1) break;
            if (there == i) {
                *again = 1;
                break;
            }
        }
    }
    team.sync();
}

// Maximum and sum of part `blockIdx % n_parts` of a row.
template <typename T, bool REST>
__global__ __launch_bounds__(256) void distill_parts(const DistillRows a) {
    __shared__ RowSums lds[4];
    extern __shared__ uint32_t distill_lds[];
    const Team<256> team = {lds};
    const int64_t row = blockIdx.x / a.n_parts;
    const int lo = (int)(blockIdx.x - row * a.n_parts) * a.part, end = min(a.V, lo + a.part), lane = threadIdx.x;
    int *index = (int *)distill_lds;
    uint32_t *bits = distill_lds + a.K;
    __shared__ int again;  // (not asked for here)
    if (REST) {
        for (int k = lane; k < a.K; k += 256) index[k] = distill_index(a, row * a.K + k);
        team.sync();
        distill_bits<T>(bits, lo, end, index, a.K, lane, team, &again);
    }
    const MaxSum r = team.join(distill_stream<T, 256, REST>((const T *)a.z + row * a.z_stride, lo, end, bits, lane, a), a.k_hi);
    if (lane == 0) a.parts[blockIdx.x] = make_float2(r.m, r.s);
}

// What the maximum and the sum of a row come from: the row itself, what distill_parts left, or a forward call's numbers
enum { FROM_ROW, FROM_PARTS, FROM_STATS };

// TPR threads take a row; HOLD elements of it stay in a thread's registers between the sum and the gradient (0: the row is read twice).  THROUGH: the gradient goes past the
// cache, which it leaves to the logits.
template <typename T, int TPR, bool REST, int FROM, int HOLD, bool THROUGH = false>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void distill_rows(const DistillRows a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR, N = Vec<T>::N, NV = HOLD ? HOLD / N : 1;
    constexpr bool FINE = sizeof(T) == 4;
    __shared__ RowSums lds[THREADS / 64];
    extern __shared__ uint32_t distill_lds[];
    if (FROM == FROM_STATS && a.leave_unit && *a.upstream == 1.0f) return;  // dz holds this gradient

    const int slot = threadIdx.x / TPR, lane = threadIdx.x % TPR;
    const Team<TPR> team = {lds};
    const int64_t block = FROM == FROM_ROW ? blockIdx.x : blockIdx.x / a.grid_parts, row = block * ROWS + slot;
    const int lo = FROM == FROM_ROW ? 0 : (int)(blockIdx.x - block * a.grid_parts) * a.part, end = FROM == FROM_ROW ? a.V : min(a.V, lo + a.part);
    const int words = REST && FROM == FROM_ROW ? bit_words(a.V) : table_places(a.K), lists = (a.K + 3) & ~3;
    double *p = (double *)((char *)distill_lds + slot * (DISTILL_ENTRY * lists + 4 * words + 8));  // (first the teacher's logits)
    int *index = (int *)(p + lists);
    float *z_list = (float *)(index + lists);
    uint32_t *bits = (uint32_t *)(z_list + lists);
    int *again = (int *)(bits + words);  // an index comes twice

    double loss = 0;
    if (row < a.rows) {
        const T *z = (const T *)a.z + row * a.z_stride;
        T *dz = a.dz ? (T *)a.dz + row * a.V : nullptr;
        const double inv_T = 1.0 / a.T;
        const float weight = a.weight ? a.weight[row] : 1.0f;

        // the list; a thread's first logit is not waited for before the pass
        float t_most = -INFINITY, z_first = -INFINITY;
        for (int k = lane; k < lists; k += TPR) {
            const int i = k < a.K ? distill_index(a, row * a.K + k) : -1;
            const float t = i < 0 ? -INFINITY : distill_logit(a, row * a.K + k);
            index[k] = i, p[k] = t;
            if (k == lane && i >= 0) z_first = (float)z[i];
            if (t > t_most || t != t) t_most = t != t ? INFINITY : t;
        }
        const double lse = REST ? (double)a.lse[row] : 0.0;
        if (lane == 0) *again = 0;
        t_most = team.max(t_most);
        team.sync();
        if (!(t_most > -INFINITY) || weight == 0.0f) {  // no entries, or no weight: no loss, no gradient
            if (dz) {
                Vec<T> zero;
#pragma unroll
                for (int e = 0; e < N; ++e) zero.v[e] = (T)0.0f;
                for (int at = lo + lane * N; at < end; at += TPR * N) Piece<T, TPR>(at, end).template store<THROUGH>(dz, zero, end);
            }
        } else {
            RowSums sums = {{-INFINITY, 0.0f}, {-INFINITY, 0.0f}, 0.0, 0.0};
            MaxSum &r = sums.pass;
            Vec<T> held[NV];
            if (FROM == FROM_PARTS) {
                for (int c = lane; c < a.n_parts; c += TPR) {
                    const float2 q = a.parts[row * a.n_parts + c];
                    if (q.x > r.m) r.s *= __builtin_amdgcn_exp2f((r.m - q.x) * a.k_hi), r.m = q.x;
                    r.s += q.y * down_to(q.x, r.m, a.k_hi);
                }
            }
            if (!REST || FROM != FROM_ROW) {
                if (dz || REST) find_again((int *)bits, index, a.K, lane, team, again);
            }
            if (FROM == FROM_ROW) {
                if (REST) distill_bits<T>(bits, 0, a.V, index, a.K, lane, team, again);
                if (HOLD) {
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) held[v] = Piece<T, TPR>((v * TPR + lane) * N, a.V).load(z, a.V);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) {
                            if (REST) Piece<T, TPR>((v * TPR + lane) * N, a.V).leave_listed(held[v], bits, 0, a.V);
                            r.m = fmaxf(r.m, most_of(held[v]));
                        }
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) r.s += exp_sum(held[v], Piece<T, TPR>((v * TPR + lane) * N, a.V).own, base_of(r.m), a);
                } else {
                    r = distill_stream<T, TPR, REST>(z, 0, a.V, bits, lane, a);
                }
            }
            team.sync();

            // the list: p without its sum (without the teacher's lse), logarithms, and the logits
            for (int k = lane; k < a.K; k += TPR) {
                const int i = index[k];
                const float zk = k == lane ? z_first : i < 0 ? -INFINITY : (float)z[i];
                const double log_p = REST ? p[k] * inv_T - lse : (p[k] - t_most) * inv_T;
                const double q = i < 0 ? 0.0 : REST ? exp_64(log_p) : (double)exp_t<true>((float)p[k] - t_most, a.k_hi, a.k_lo);
                z_list[k] = zk, p[k] = q;
                sums.p += q;
                if (q != 0) sums.a += q * (log_p - zk * inv_T);
                if (REST && FROM != FROM_STATS) {
                    bool before = false;
                    if (*again)
                        for (int l = 0; l < k; ++l) before |= index[l] == i;
                    if (i >= 0 && !before) {
                        if (zk > sums.list.m) sums.list.s *= exp_t<true>(sums.list.m - zk, a.k_hi, a.k_lo), sums.list.m = zk;
                        sums.list.s += exp_t<true>(zk - base_of(sums.list.m), a.k_hi, a.k_lo);
                    }
                }
            }
            sums = team.join(sums, a.k_hi);

            // m, a of the pass and M, b of the list
            float m, pass, M, list;
            if (FROM == FROM_STATS) {
                const float4 s = a.stats[row];
                m = s.x, pass = s.y, M = s.z, list = s.w;
            } else {
                const float most = REST ? fmaxf(r.m, sums.list.m) : r.m;
                m = base_of(r.m), M = base_of(most);
                float total = r.s, p_rest = 0;
                if (REST) {
                    // (a side that has nothing has no maximum either)
                    const float down = r.s == 0.0f ? 0.0f : exp_t<true>(m - M, a.k_hi, a.k_lo);
                    total = r.s * down + (sums.list.s == 0.0f ? 0.0f : sums.list.s * exp_t<true>(sums.list.m - M, a.k_hi, a.k_lo));
                    if (r.s > 0.0f) p_rest = (float)fmax(0.0, 1.0 - sums.p);
                    const float P = (float)sums.p + p_rest;
                    pass = r.s == 0.0f ? 0.0f : P * down / total - p_rest / r.s;
                    list = P / total;
                } else {
                    pass = list = 1.0f / total;
                }
                if (threadIdx.x - slot * TPR < 64) {  // (one wavefront)
                    if (REST) {
                        loss = sums.a + sums.p * (M * inv_T + log_64(total));
                        if (p_rest > 0) loss += p_rest * (log_64((double)p_rest * total / r.s) + ((double)M - m) * inv_T);
                    } else {
                        loss = sums.a / sums.p + log_64(total / sums.p) + M * inv_T;
                    }
                    loss *= weight * a.scale;
                    if (a.stats && lane == 0 && lo == 0) a.stats[row] = make_float4(m, pass, M, list);
                }
            }

            if (dz) {
                const float c = (float)(weight * a.scale * inv_T) * (FROM == FROM_STATS ? *a.upstream : 1.0f), ca = c * pass;
                auto gradient = [&](const Vec<T> &v, int at) {
                    Vec<T> o;
#pragma unroll
                    for (int e = 0; e < N; ++e) o.v[e] = (T)(ca * exp_t<FINE>((float)v.v[e] - m, a.k_hi, a.k_lo));
                    Piece<T, TPR>(at, end).template store<THROUGH>(dz, o, end);
                };
                if (HOLD) {
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (v * TPR * N < a.V) gradient(held[v], (v * TPR + lane) * N);
                } else {
                    for (int at = lo + lane * N; at < end; at += AHEAD * TPR * N) {
                        Vec<T> v[AHEAD];
#pragma unroll
                        for (int k = 0; k < AHEAD; ++k) v[k] = Piece<T, TPR>(at + k * TPR * N, end).load(z, end);
#pragma unroll
                        for (int k = 0; k < AHEAD; ++k) gradient(v[k], at + k * TPR * N);
                    }
                }
                // the list's entries, over what the pass wrote there
                __threadfence_block();
                team.sync();
                const float one = REST ? 1.0f : 1.0f / (float)sums.p;
                for (int k = lane; k < a.K; k += TPR) {
                    const int i = index[k];
                    if (i < lo || i >= end) continue;
                    double sum = p[k];
                    if (*again) {  // (in the list's order, so that all of them write the same)
                        sum = 0;
                        for (int l = 0; l < a.K; ++l)
                            if (index[l] == i) sum += p[l];
                    }
                    dz[i] = (T)(c * (list * exp_t<true>(z_list[k] - M, a.k_hi, a.k_lo) - (float)sum * one));
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
        if (threadIdx.x == 0) {
            if (a.loss) *a.loss = (float)loss;  // (the only one)
            else a.losses[block] = loss;
        }
    }
}

__global__ __launch_bounds__(1024) void distill_sum(const double *__restrict__ losses, int64_t n, float *__restrict__ loss) {
    __shared__ double lds[16];
    double s = 0;
    for (int64_t k = threadIdx.x; k < n; k += 1024) s += losses[k];
    s = team_sum(s, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = team_sum(lds[threadIdx.x & 15], 16);
    if (threadIdx.x == 0) *loss = (float)s;
}

namespace {

constexpr int SPLIT_ROWS = 128;   // rows from which on a row has a workgroup to itself (200 x 131072 bfloat16 with gradient: 37 us, in three parts 44)
constexpr int SPLIT_PART = 4096;  // entries of a part, at least
constexpr int SPLIT_TERMS = 64;   // terms that a thread adds up one after the other, at most (1000 x 262144 float32 with gradient 556 us, four entries more, in parts, 656)

struct DistillPlan {
    int tpr, hold;      // threads per row, elements held
    int n_parts, part;  // of a row
    int64_t blocks;     // sums of losses
};

// us for the loss with its gradient (without the teacher's lse), and for the loss alone:
// * 8 and 16 threads: a row costs its list, whatever its length, and a wavefront takes eight or four lists at once (100000 x 100 float32: 16 threads 32 and 22, 64 threads
//   86 and 66).
// * A wavefront needs no barrier and has the most rows in flight, but takes long for a long row (16000 x 4000 bfloat16: 65 and 34, 256 threads 81 and 62; 8192 x 10000
//   float32: 175 and 59, 256 threads 127 and 67; 1000 x 4000 bfloat16: 15 and 11, 256 threads 12 and 11).
// * Rows that are held save the second read, and cost registers that others' loads would need: up to 64 elements a thread (8192 x 10000 float32: 127, read twice 155;
//   4096 x 32000 bfloat16 in 128 a thread: 145, read twice 128).
// * Rows that are read twice find what the first read left in the card's 256 MB cache while those in flight are a part of it: 64 KB a row with eight
//   workgroups a compute unit, 256 KB with four, two beyond (4096 x 131072 bfloat16: 256 threads 628, 512 507, 1024 484, and with the teacher's lse, whose
//   list a smaller workgroup waits less for, 622, 521, 650; float32 1242, 1151, 976).  The loss alone reads once (227, 260 and 340 with the lse).
DistillPlan distill_plan(int64_t rows, int V, int K, bool rest, int size, bool gradient) {
    DistillPlan p = {};
    const int64_t bytes = (int64_t)V * size;
    if (V <= 64 && K <= 64) p.tpr = 8, p.hold = 8;
    else if (V <= 256 && K <= 64) p.tpr = 16, p.hold = 16;
    else if (V <= 2048 && K <= 512) p.tpr = 64, p.hold = 32;
    else if (rows >= 4096 && K <= 512 && bytes <= (gradient ? 16 << 10 : 64 << 10)) p.tpr = 64, p.hold = 0;
    else if (gradient && V <= 16384) p.tpr = 256, p.hold = 64;
    else p.tpr = !gradient || bytes <= 64 << 10 ? 256 : bytes <= 256 << 10 ? 512 : 1024, p.hold = 0;
    p.n_parts = 1, p.part = V;
    int64_t parts = 1;
    if (rows < SPLIT_ROWS && V >= 2 * SPLIT_PART) parts = (512 + rows - 1) / rows;
    if (parts > V / SPLIT_PART) parts = V / SPLIT_PART;
    if (rest && parts < (V + DISTILL_BITS - 1) / DISTILL_BITS) parts = (V + DISTILL_BITS - 1) / DISTILL_BITS;
    const int64_t longest = SPLIT_TERMS * (16 / size);  // entries of a thread
    if ((parts > 1 || V > longest * p.tpr) && parts < (V + 256 * longest - 1) / (256 * longest)) parts = (V + 256 * longest - 1) / (256 * longest);
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
    if (rows < 0 || V < 1 || K < 1 || !(T >= 1e-30 && T <= 1e30)) return fail(HGQ_ERR_ARG, "%s: rows %lld, vocabulary %lld, list %lld, temperature %g", what, (long long)rows, (long long)V, (long long)K, T);
    if (type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16 || t_type < HGQ_TYPE_F32 || t_type > HGQ_TYPE_F16) return fail(HGQ_ERR_ARG, "%s: unknown type", what);
    if (index_bytes != 4 && index_bytes != 8) return fail(HGQ_ERR_ARG, "%s: indices of %d bytes", what, index_bytes);
    if (K > DISTILL_LIST) return fail(HGQ_ERR_UNSUPPORTED, "%s: a list of %lld entries, at most %d", what, (long long)K, DISTILL_LIST);
    // (teams of eight are the only ones whose accesses may be cut, and the lists of 32 rows have to fit)
    if (K > 64 && V < 8) return fail(HGQ_ERR_UNSUPPORTED, "%s: a list of %lld entries, at most 64 of a vocabulary of %lld", what, (long long)K, (long long)V);
    if (V > 1 << 30 || rows > (int64_t)1 << 40) return fail(HGQ_ERR_UNSUPPORTED, "%s: %lld rows of %lld entries", what, (long long)rows, (long long)V);
    return HGQ_OK;
}

int64_t lds_of(const DistillRows &a, int tpr, bool bits, int entries) {
    return (int64_t)(tpr < 256 ? 256 / tpr : 1) * (DISTILL_ENTRY * ((a.K + 3) & ~3) + 4 * (bits ? bit_words(entries) : table_places(a.K)) + 8);
}

template <typename T, int TPR, bool REST, int FROM, int HOLD, bool THROUGH = false>
int launch(const DistillRows &a, int64_t blocks, int64_t lds, hipStream_t st, const char *what) {
    constexpr int threads = TPR > 256 ? TPR : 256;
    if (blocks * threads > 0xffffffffLL) return fail(HGQ_ERR_UNSUPPORTED, "%s: too many rows", what);
    hipLaunchKernelGGL((distill_rows<T, TPR, REST, FROM, HOLD, THROUGH>), dim3((unsigned)blocks), dim3(threads), (size_t)lds, st, a);
    return check_launch(what);
}

template <typename T, bool REST>
int forward(DistillRows a, const DistillPlan &p, float *loss, hipStream_t st) {
    const char *what = "hgq_distill_topk_fwd";
    a.n_parts = p.n_parts, a.part = p.part, a.loss = p.blocks == 1 ? loss : nullptr;
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
        const bool through = a.dz && a.rows * a.V * (int64_t)sizeof(T) * 2 > (int64_t)256 << 20;  // logits and gradient are more than the card's cache
        rc = p.tpr == 8      ? launch<T, 8, REST, FROM_ROW, 8>(a, p.blocks, lds, st, what)
             : p.tpr == 16  ? launch<T, 16, REST, FROM_ROW, 16>(a, p.blocks, lds, st, what)
             : p.tpr == 64  ? p.hold ? launch<T, 64, REST, FROM_ROW, 32>(a, p.blocks, lds, st, what) : launch<T, 64, REST, FROM_ROW, 0>(a, p.blocks, lds, st, what)
             : p.tpr == 256 ? p.hold      ? launch<T, 256, REST, FROM_ROW, 64>(a, p.blocks, lds, st, what)
                              : through ? launch<T, 256, REST, FROM_ROW, 0, true>(a, p.blocks, lds, st, what)
                                        : launch<T, 256, REST, FROM_ROW, 0>(a, p.blocks, lds, st, what)
             : p.tpr == 512 ? through ? launch<T, 512, REST, FROM_ROW, 0, true>(a, p.blocks, lds, st, what) : launch<T, 512, REST, FROM_ROW, 0>(a, p.blocks, lds, st, what)
             : through      ? launch<T, 1024, REST, FROM_ROW, 0, true>(a, p.blocks, lds, st, what)
                            : launch<T, 1024, REST, FROM_ROW, 0>(a, p.blocks, lds, st, what);
    }
    if (rc || p.blocks == 1) return rc;
    hipLaunchKernelGGL(distill_sum, dim3(1), dim3(1024), 0, st, (const double *)a.losses, p.blocks, loss);
    return check_launch(what);
}

template <typename T, bool REST>
int backward(DistillRows a, const DistillPlan &p, hipStream_t st) {
    const char *what = "hgq_distill_topk_bwd";
    a.grid_parts = p.n_parts, a.part = p.part;
    const int64_t lds = lds_of(a, p.tpr, false, 0), blocks = p.blocks * p.n_parts;
    return p.tpr == 16    ? launch<T, 16, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 8   ? launch<T, 8, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 64  ? launch<T, 64, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 256 ? launch<T, 256, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
           : p.tpr == 512 ? launch<T, 512, REST, FROM_STATS, 0>(a, blocks, lds, st, what)
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
    int most = 1;
    for (int kind = 0; kind < 4; ++kind) most = std::max(most, distill_plan(rows, (int)V, (int)K, rest, kind & 1 ? 2 : 4, kind & 2).n_parts);
    return 2 * rows + (most > 1 ? 2 * rows * most : 0);  // (a sum for each row, at most)
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
    const DistillPlan p = distill_plan(rows, (int)V, (int)K, lse != nullptr, type == HGQ_TYPE_F32 ? 4 : 2, dz != nullptr);
    a.stats = (float4 *)stats, a.dz = dz, a.losses = (double *)workspace, a.parts = (float2 *)(workspace + 2 * rows);
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
    const DistillPlan p = distill_plan(rows, (int)V, (int)K, lse != nullptr, type == HGQ_TYPE_F32 ? 4 : 2, true);
    hipStream_t st = (hipStream_t)stream;
    if (lse) return type == HGQ_TYPE_F32 ? backward<float, true>(a, p, st) : type == HGQ_TYPE_BF16 ? backward<__bf16, true>(a, p, st) : backward<_Float16, true>(a, p, st);
    return type == HGQ_TYPE_F32 ? backward<float, false>(a, p, st) : type == HGQ_TYPE_BF16 ? backward<__bf16, false>(a, p, st) : backward<_Float16, false>(a, p, st);
}
