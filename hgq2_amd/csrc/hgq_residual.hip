// What stands between two blocks of a network: the norm behind the first, its gate, the residual sum and the norm ahead of the second.
// Rows of C channels, norm(v) = v / sqrt(mean(v^2) + eps):
//     n = norm(u);   b = scale act(gate) n post;   y = x + b;   h = norm(y) pre               (act: none, or 1 / (1 + exp(-gate)))
// Backward, given dy and dh, with m = norm(y), e = dh pre and r_u, r_y the factors of both norms:
//     dx = dy + r_y (e - m mean(e m));   dn = dx scale act(gate) post;   du = r_u (dn - n mean(dn n))
//     dpre = sum dh m,  dpost = sum dx scale act(gate) n  over rows;   dgate = dx scale n post act'(gate)
// A gate has an element for each of x, or one row for P rows (a sample's positions): its gradient is then a sum over them.  Without u: y = x.
//
// Bound by memory.  One pass each way: a row's elements stay in registers, eight a thread, while a team of as many threads as the row needs
// forms both means; the backward pass forms y again from x (which costs the bytes that y would, and keeps what y's rounding drops).  Sums over rows stay
// in registers while a workgroup goes from row to row, and leave in slices, at least one a workgroup and one for 64 rows of a thread, which are joined in 64 bits in a fixed order.
#include <algorithm>
#include <type_traits>

#include "hgq_host.h"
#include "hgq_vector.h"

namespace hgq {

constexpr int RES_HELD = 8;     // elements of a row in a thread
constexpr int RES_WIDEST = 8192;  // channels up to which 1024 threads hold a row

struct ResidualRows {
    const void *x, *u, *gate, *dy, *dh;
    const float *post, *pre;
    void *y, *h, *dx, *du, *dgate;
    float *r_u, *r_y;
    float *slices;       // [..][2][C]: dpost, dpre; a workgroup's j-th one is j workgroups' number behind its first
    float *gate_slices;  // [units][C], or null: dgate is written as it is formed
    int64_t step_samples, step_rows;         // of a workgroup's step over rows, in samples and rows
    int64_t samples;                         // rows of a gate for P rows
    int64_t rows, P, units, per_unit, cuts;  // rows; of a gate's row; what a workgroup takes at a time, its rows; units of a sample
    int C, tpr, act, by_sample, run;  // run: units that a workgroup adds up in a slice
    float scale, eps, inv_c;
};

// The threads of a row: neighbouring lanes of a wavefront, or (WIDE) a workgroup of as many wavefronts as it needs.  Sums of a workgroup take turns with two places in LDS:
// whoever writes one again is behind the barrier of the sum between.
template <bool WIDE>
struct RowTeam {
    int tpr;
    float (*lds)[16];
    int turn, slots;  // wavefronts, up to the next power of two
    __device__ __forceinline__ RowTeam(int tpr, float (*lds)[16]) : tpr(tpr), lds(lds), turn(0), slots(1) {
        if (!WIDE) return;
        while (slots < tpr >> 6) slots *= 2;
        if (threadIdx.x < 16 && threadIdx.x >= tpr >> 6) lds[0][threadIdx.x] = lds[1][threadIdx.x] = 0.0f;  // (visible behind the first sum's barrier)
    }
    __device__ __forceinline__ float sum(float v) {
        if (!WIDE) return team_sum(v, tpr);
        v = team_sum(v, 64);
        float *at = lds[turn ^= 1];
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        return team_sum(at[threadIdx.x & (slots - 1)], slots);
    }
};

// (the hardware's root, a unit in the last place off, and a product with 1 / C: with the root refined to half a unit float32 outputs and gradients are no nearer to 64 bits,
// their errors' mean squares within a tenth either way.  Rounded ones take 1531 x 30 x 333 float16 with a gate forward 33.3 us, these 30.7, 32768 x 1536 bfloat16 91.8 and 89.2; backward no
// difference.  Times here and below are GPU times of whole calls, joins included, with the same inputs each time unless they are said to be read anew.)
__device__ __forceinline__ float norm_factor(float sum, float inv_c, float eps) {
    const float square = sum * inv_c + eps;
    const bool tiny = square < 0x1p-100f;  // (without an epsilon: the root takes numbers below fp32's normal ones for zero)
    return __builtin_amdgcn_rsqf(tiny ? square * 0x1p100f : square) * (tiny ? 0x1p50f : 1.0f);
}

// (the hardware's exponential and reciprocal, a unit each, and an exponent off by |g| 2^-24, which the sigmoid's own slope makes less: 16-bit types do not show it, and float32
// gradients are nearer to 64 bits than elementary operations get them)
__device__ __forceinline__ float opened(float g, int act) { return act ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269502f)) : g; }

// A thread's eight elements of a row.  A row's last access ends with the row: its first elements are the neighbour's again, which are left out of sums and written
// twice.  TINY: rows of less than one access.
template <typename T, bool TINY>
struct Held {
    static constexpr int N = Vec<T>::N, NV = RES_HELD / N;
    struct Raw {
        u32x4 v[NV];
    };
    int at[NV], own[NV];  // this thread's columns, and which of the first ones are the neighbour's
    int C;
    __device__ __forceinline__ Held(int lane, int tpr, int channels) : C(channels) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int wanted = (v * tpr + lane) * N;
            at[v] = TINY ? wanted : min(wanted, C - N), own[v] = min(N, wanted - at[v]);
        }
    }
    __device__ __forceinline__ Raw ask(const T *row) const {
        Raw r;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (TINY) r.v[v] = __builtin_bit_cast(u32x4, load_part(row + at[v], C - at[v], (T)0.0f));
            else r.v[v] = load_words(row + at[v]);
        }
        return r;
    }
    __device__ __forceinline__ void take(float *f, const Raw &r) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Vec<T> w = __builtin_bit_cast(Vec<T>, r.v[v]);
#pragma unroll
            for (int e = 0; e < N; ++e) f[v * N + e] = (float)w.v[e];
        }
    }
    __device__ __forceinline__ void store(T *row, const float *f) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            Vec<T> r;
#pragma unroll
            for (int e = 0; e < N; ++e) r.v[e] = (T)f[v * N + e];
            if (TINY) store_part(row + at[v], r, C - at[v]);
            else if (own[v] < N) store_vec(row + at[v], r);
        }
    }
    // the sum of products over this thread's own elements
    __device__ __forceinline__ float dot(const float *f, const float *g) const {
        float s = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < N; ++e) s += e < own[v] ? 0.0f : f[v * N + e] * g[v * N + e];
        return s;
    }
    __device__ __forceinline__ bool mine(int v, int e) const { return e >= own[v] && at[v] + e < C; }
    __device__ __forceinline__ void vector(float *f, const float *p, float scale) const {  // of channels, times `scale`
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < N; ++e) f[v * N + e] = p ? p[TINY ? min(at[v] + e, C - 1) : at[v] + e] : 1.0f;
#pragma unroll
        for (int e = 0; e < RES_HELD; ++e) f[e] *= scale;
    }
};

// rows of less than one access; of a wavefront (257 .. 512 channels), whose addresses are then scalars (1531 x 30 x 333 float16 backward, read anew: 65 -> 62 us with a gate, 56 -> 53
// without; forward 32 -> 31 and 26 -> 25); all others
enum { TINY_ROWS, WAVE_ROWS, ROWS };
enum { NO_UPDATE, NO_GATE, GATED, GATED_SAMPLES };  // the last: one row of a gate for P rows

template <typename T, int KIND, int THREADS, int FORM>
__global__ __launch_bounds__(THREADS) void residual_fwd(const ResidualRows a) {
    constexpr bool WIDE = THREADS > 256, TINY = FORM == TINY_ROWS;
    __shared__ float lds[2][16];
    using H = Held<T, TINY>;
    const int tpr = FORM == WAVE_ROWS ? 64 : a.tpr, teams = WIDE ? 1 : 256 / tpr;
    const int slot = WIDE ? 0 : FORM == WAVE_ROWS ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / tpr, lane = WIDE ? threadIdx.x : threadIdx.x & (tpr - 1);
    const H held(lane, tpr, a.C);
    RowTeam<WIDE> team(tpr, lds);
    float post[RES_HELD], pre[RES_HELD];
    if (KIND != NO_UPDATE) held.vector(post, a.post, a.scale);
    held.vector(pre, a.pre, 1.0f);
    const int64_t step = (int64_t)gridDim.x * teams;
    int64_t row = (int64_t)blockIdx.x * teams + slot, sample = 0, position = 0;
    if (KIND == GATED_SAMPLES) sample = row / a.P, position = row - sample * a.P;
    typename H::Raw x_raw, u_raw, g_raw;
    auto ask = [&](int64_t k) {
        const int64_t base = min(k, a.rows - 1) * a.C;
        x_raw = held.ask((const T *)a.x + base);
        if (KIND != NO_UPDATE) u_raw = held.ask((const T *)a.u + base);
        if (KIND >= GATED) g_raw = held.ask((const T *)a.gate + (KIND == GATED_SAMPLES ? min(sample, a.samples - 1) * a.C : base));
    };
    ask(row);
    for (; row < a.rows; row += step) {
        const int64_t base = row * a.C;
        float y[RES_HELD], u[RES_HELD], g[RES_HELD];
        held.take(y, x_raw);
        if (KIND != NO_UPDATE) held.take(u, u_raw);
        if (KIND >= GATED) held.take(g, g_raw);
        if (KIND == GATED_SAMPLES) {
            sample += a.step_samples, position += a.step_rows;
            if (position >= a.P) position -= a.P, ++sample;
        }
        ask(row + step);  // on its way while this row is worked on
        if (KIND != NO_UPDATE) {
            const float r_u = norm_factor(team.sum(held.dot(u, u)), a.inv_c, a.eps);
#pragma unroll
            for (int e = 0; e < RES_HELD; ++e) {
                float b = u[e] * r_u * post[e];
                if (KIND >= GATED) b *= opened(g[e], a.act);
                y[e] += b;
            }
            if (a.r_u && lane == 0) a.r_u[row] = r_u;
            held.store((T *)a.y + base, y);
        }
        const float r_y = norm_factor(team.sum(held.dot(y, y)), a.inv_c, a.eps);
        if (a.r_y && lane == 0) a.r_y[row] = r_y;
#pragma unroll
        for (int e = 0; e < RES_HELD; ++e) y[e] *= r_y * pre[e];
        held.store((T *)a.h + base, y);
    }
}

template <typename T, int KIND, int THREADS, int FORM>
__global__ __launch_bounds__(THREADS) void residual_bwd(const ResidualRows a) {
    constexpr bool WIDE = THREADS > 256, TINY = FORM == TINY_ROWS;
    __shared__ float lds[2][16];
    __shared__ float joined[WIDE ? 1 : 256 * RES_HELD];
    using H = Held<T, TINY>;
    const int tpr = FORM == WAVE_ROWS ? 64 : a.tpr, teams = WIDE ? 1 : 256 / tpr;
    const int slot = WIDE ? 0 : FORM == WAVE_ROWS ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / tpr, lane = WIDE ? threadIdx.x : threadIdx.x & (tpr - 1);
    const H held(lane, tpr, a.C);
    RowTeam<WIDE> team(tpr, lds);
    // What a thread keeps from row to row of its columns' post, pre, dpost and dpre.  With 1024 threads, which have 128 registers each, it lies in LDS, where no other
    // thread looks at it (8192 x 8192 bfloat16, a gate like x: 233 us instead of 330 with 32 registers spilled; float32 with a gate still spills 2, with one for samples 10).
    constexpr bool STASH = THREADS == 1024 && KIND != NO_UPDATE;
    __shared__ float4 stash[STASH ? 4 : 1][RES_HELD / 4][STASH ? THREADS : 1];
    enum { POST, PRE, DPOST, DPRE };
    float kept[4][RES_HELD] = {}, dgate[RES_HELD] = {};
    auto recall = [&](int which, float *f) {
#pragma unroll
        for (int q = 0; q < RES_HELD / 4; ++q) {
            if (STASH) {
                const float4 v = stash[which][q][threadIdx.x];
                f[4 * q] = v.x, f[4 * q + 1] = v.y, f[4 * q + 2] = v.z, f[4 * q + 3] = v.w;
            } else {
#pragma unroll
                for (int e = 4 * q; e < 4 * q + 4; ++e) f[e] = kept[which][e];
            }
        }
    };
    auto keep = [&](int which, const float *f) {
#pragma unroll
        for (int q = 0; q < RES_HELD / 4; ++q) {
            if (STASH) {
                stash[which][q][threadIdx.x] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
            } else {
#pragma unroll
                for (int e = 4 * q; e < 4 * q + 4; ++e) kept[which][e] = f[e];
            }
        }
    };
    {
        float f[RES_HELD] = {};
        keep(DPOST, f), keep(DPRE, f);
        if (KIND != NO_UPDATE) held.vector(f, a.post, a.scale), keep(POST, f);
        held.vector(f, a.pre, 1.0f), keep(PRE, f);
    }

    // one row of channels from the teams' sums, in order
    auto leave = [&](const float *f, auto *out) {
        using Out = std::remove_reference_t<decltype(*out)>;
        if (WIDE) {
#pragma unroll
            for (int v = 0; v < H::NV; ++v)
#pragma unroll
                for (int e = 0; e < H::N; ++e)
                    if (held.mine(v, e)) out[held.at[v] + e] = (Out)f[v * H::N + e];
            return;
        }
        int at = slot * a.C;
        asm("" : "+v"(at));  // (places in LDS are worked out here, not kept in registers through the rows)
        __syncthreads();
#pragma unroll
        for (int v = 0; v < H::NV; ++v)
#pragma unroll
            for (int e = 0; e < H::N; ++e)
                if (held.mine(v, e)) joined[at + held.at[v] + e] = f[v * H::N + e];
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += 256) {
            double s = 0;  // (up to 256 teams)
#pragma unroll 8  // (one read after the other takes 2 us of a launch)
            for (int t = 0; t < teams; ++t) s += joined[t * a.C + c];
            out[c] = (Out)(float)s;
        }
    };

    // where the workgroup stands: rows r .. r + teams - 1 of a unit's rows below r1
    struct Step {
        int64_t unit, sample, r, r1;
    };
    auto enter = [&](int64_t unit) {
        const int64_t sample = KIND == GATED_SAMPLES ? unit / a.cuts : 0, r0 = sample * a.P + (unit - sample * a.cuts) * a.per_unit;
        return Step{unit, sample, r0, min(min(r0 + a.per_unit, (sample + 1) * a.P), a.rows)};
    };
    typename H::Raw x_raw, u_raw, g_raw, dy_raw = {}, dh_raw = {};
    float r_u_next = 0, r_y_next = 0;
    auto ask = [&](const Step &k) {
        const int64_t row = min(k.r + slot, a.rows - 1), base = row * a.C;
        x_raw = held.ask((const T *)a.x + base);
        if (KIND != NO_UPDATE) u_raw = held.ask((const T *)a.u + base);
        if (KIND >= GATED) g_raw = held.ask((const T *)a.gate + (KIND == GATED_SAMPLES ? min(k.sample, a.samples - 1) * a.C : base));
        if (a.dy) dy_raw = held.ask((const T *)a.dy + base);
        if (a.dh) dh_raw = held.ask((const T *)a.dh + base);
        if (KIND != NO_UPDATE) r_u_next = a.r_u[row];
        r_y_next = a.r_y[row];
    };
    // Where a gate's row stands for a unit's rows, they add up dx n alone: dgate and dpost are that times factors of the unit.
    float open[RES_HELD];
    bool first = true;
    int slice = blockIdx.x;
    int taken = 0;  // units in this slice
    Step k = enter(blockIdx.x);
    ask(k);
    while (k.unit < a.units) {  // a slice
        bool last;
        do {
            float x[RES_HELD], n[RES_HELD], g[RES_HELD], dy[RES_HELD], dh[RES_HELD];
            held.take(x, x_raw);
            if (KIND != NO_UPDATE) held.take(n, u_raw);
            if (KIND == GATED) held.take(g, g_raw);
            if (KIND == GATED_SAMPLES && first) {
                held.take(open, g_raw);
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) open[e] = opened(open[e], a.act);
            }
            held.take(dy, dy_raw);
            held.take(dh, dh_raw);
            const float r_u = r_u_next, r_y = r_y_next;
            const Step now = k;
            last = k.r + teams >= k.r1;
            first = last;
            if (last) k = enter(k.unit + gridDim.x);
            else k.r += teams;
            ask(k);  // on its way while these rows are worked on
            const bool there = now.r + slot < now.r1;
            const int64_t base = (now.r + slot) * a.C;
            if (!there) {
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) dy[e] = dh[e] = 0;
            }
            if (KIND != NO_UPDATE) {
                float post[RES_HELD];
                recall(POST, post);
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) {
                    n[e] *= r_u;
                    float b = n[e] * post[e];
                    if (KIND == GATED) open[e] = opened(g[e], a.act);
                    if (KIND >= GATED) b *= open[e];
                    x[e] += b;
                }
            }
            float s = 0;
            if (a.dh) {
                float pre[RES_HELD], dpre[RES_HELD];
                recall(PRE, pre), recall(DPRE, dpre);
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) {
                    x[e] *= r_y;  // m
                    if (there) dpre[e] += dh[e] * x[e];
                    dh[e] *= pre[e];
                }
                keep(DPRE, dpre);
                s = team.sum(held.dot(dh, x)) * a.inv_c;
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) dy[e] += r_y * (dh[e] - x[e] * s);
            }
            if (a.dx && there) held.store((T *)a.dx + base, dy);
            if (KIND != NO_UPDATE) {
                float dn[RES_HELD], post[RES_HELD], dpost[RES_HELD];
                recall(POST, post);
                if (KIND != GATED_SAMPLES) recall(DPOST, dpost);
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) {
                    const float db = KIND >= GATED ? dy[e] * open[e] : dy[e];
                    if (there && KIND == GATED_SAMPLES) dgate[e] += dy[e] * n[e];
                    if (there && KIND != GATED_SAMPLES) dpost[e] += db * n[e];
                    dn[e] = db * post[e];
                    if (KIND == GATED) {
                        open[e] = dy[e] * (n[e] * post[e]) * (a.act ? open[e] * (1.0f - open[e]) : 1.0f);
                    }
                }
                if (KIND != GATED_SAMPLES) keep(DPOST, dpost);
                if (KIND == GATED && a.dgate && there) held.store((T *)a.dgate + base, open);
                if (a.du) {
                    s = team.sum(held.dot(dn, n)) * a.inv_c;
#pragma unroll
                    for (int e = 0; e < RES_HELD; ++e) dn[e] = r_u * (dn[e] - n[e] * s);
                    if (there) held.store((T *)a.du + base, dn);
                }
                if (KIND == GATED_SAMPLES && last) {
                    recall(POST, post), recall(DPOST, dpost);
#pragma unroll
                    for (int e = 0; e < RES_HELD; ++e) {
                        dpost[e] += dgate[e] * open[e];
                        dgate[e] *= post[e] * (a.act ? open[e] * (1.0f - open[e]) : 1.0f);
                    }
                    keep(DPOST, dpost);
                    if (!a.dgate) {
                    } else if (a.gate_slices) leave(dgate, a.gate_slices + now.unit * a.C);
                    else leave(dgate, (T *)a.dgate + now.sample * a.C);
#pragma unroll
                    for (int e = 0; e < RES_HELD; ++e) dgate[e] = 0;
                }
            }
        } while (!last || (++taken < a.run && k.unit < a.units));
        taken = 0;
        if (a.slices) {
            float *out = a.slices + (int64_t)slice * 2 * a.C, f[RES_HELD], none[RES_HELD] = {};
            if (KIND != NO_UPDATE) {
                recall(DPOST, f);
#pragma unroll
                for (int e = 0; e < RES_HELD; ++e) f[e] *= a.scale;
                leave(f, out);
                keep(DPOST, none);
            }
            recall(DPRE, f);
            leave(f, out + a.C);
            keep(DPRE, none);
            slice += gridDim.x;
        }
    }
}

// Rows of more channels than a workgroup holds: read again for each of the means, ANY columns of a thread at a time (all their loads ahead of their stores: 4000 x 12000 bfloat16
// 201 and 442 us, one by one 250 and 875); sums over rows in the workgroup's own slices, means' sums in 64 bits beyond four columns.
constexpr int ANY = 4;

template <typename T>
struct AnyRow {
    const ResidualRows &a;
    int64_t base, gate_base;
    float r_u;
    struct Columns {  // n = norm(u) (without post), open = act(gate), post with the scale
        float y[ANY], n[ANY], open[ANY], post[ANY], pre[ANY], dy[ANY], dh[ANY];
    };
    __device__ __forceinline__ int column(int c, int k) const { return min(c + 1024 * k, a.C - 1); }
    // (what there is not is read from x: elements of 16 bits loaded in a branch would be waited for there)
    __device__ __forceinline__ void one(float *f, const void *from, int64_t at, int c) const {
        const T *p = from ? (const T *)from + at : (const T *)a.x + base;
        T v[ANY];
#pragma unroll
        for (int k = 0; k < ANY; ++k) v[k] = p[column(c, k)];
#pragma unroll
        for (int k = 0; k < ANY; ++k) f[k] = from ? (float)v[k] : 0.0f;
    }
    __device__ __forceinline__ void factor(float *f, const float *from, int c) const {
#pragma unroll
        for (int k = 0; k < ANY; ++k) f[k] = from ? from[column(c, k)] : 1.0f;
    }
    // the sum of products over these columns: a thread adds up such sums in 64 bits (it has as many as a row is long)
    __device__ __forceinline__ float dot(const float *f, const float *g, int c) const {
        float s = 0;
#pragma unroll
        for (int k = 0; k < ANY; ++k) s += c + 1024 * k < a.C ? f[k] * g[k] : 0.0f;
        return s;
    }
    __device__ __forceinline__ Columns take(int c, bool gradients) const {
        Columns v;
        one(v.y, a.x, base, c), one(v.n, a.u, base, c), one(v.open, a.gate, gate_base, c);
        factor(v.post, a.post, c), factor(v.pre, a.pre, c);
        if (gradients) one(v.dy, a.dy, base, c), one(v.dh, a.dh, base, c);
#pragma unroll
        for (int k = 0; k < ANY; ++k) {
            v.n[k] *= r_u, v.post[k] *= a.scale, v.open[k] = a.gate ? opened(v.open[k], a.act) : 1.0f;
            v.y[k] += v.n[k] * v.post[k] * v.open[k];  // (without an update n is zero)
        }
        return v;
    }
    // dx, with m = norm(y)
    __device__ __forceinline__ float through(const Columns &v, int k, float r_y, float s1) const { return v.dy[k] + r_y * (v.dh[k] * v.pre[k] - v.y[k] * r_y * s1); }
};

template <typename T>
__global__ __launch_bounds__(1024) void residual_fwd_any(const ResidualRows a) {
    __shared__ float lds[2][16];
    RowTeam<true> team(1024, lds);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        AnyRow<T> r = {a, row * a.C, a.by_sample ? row / a.P * a.C : row * a.C, 0.0f};
        double s = 0;
        if (a.u) {
            for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
                float u[ANY];
                r.one(u, a.u, r.base, c);
                s += r.dot(u, u, c);
            }
            r.r_u = norm_factor(team.sum((float)s), a.inv_c, a.eps);
            s = 0;
        }
        for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
            const auto v = r.take(c, false);
            s += r.dot(v.y, v.y, c);
        }
        const float r_y = norm_factor(team.sum((float)s), a.inv_c, a.eps);
        for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
            const auto v = r.take(c, false);
#pragma unroll
            for (int k = 0; k < ANY; ++k) {
                const int at = c + 1024 * k;
                if (at >= a.C) break;
                if (a.u) ((T *)a.y)[r.base + at] = (T)v.y[k];
                ((T *)a.h)[r.base + at] = (T)(v.y[k] * (r_y * v.pre[k]));
            }
        }
        if (threadIdx.x == 0) {
            if (a.r_u) a.r_u[row] = r.r_u;
            if (a.r_y) a.r_y[row] = r_y;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void residual_bwd_any(const ResidualRows a) {
    __shared__ float lds[2][16];
    RowTeam<true> team(1024, lds);
    int slice = blockIdx.x;
    int taken = 0;  // units in this slice
    for (int64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        if (taken == a.run) taken = 0, slice += gridDim.x;
        float *dpost = a.slices ? a.slices + (int64_t)slice * 2 * a.C : nullptr, *dpre = dpost ? dpost + a.C : nullptr;
        const int64_t sample = unit / a.cuts, r0 = sample * a.P + (unit - sample * a.cuts) * a.per_unit, r1 = min(min(r0 + a.per_unit, (sample + 1) * a.P), a.rows);
        float *dgate = a.by_sample && a.dgate ? a.gate_slices + unit * a.C : nullptr;
        for (int64_t row = r0; row < r1; ++row) {
            const AnyRow<T> r = {a, row * a.C, a.by_sample ? sample * a.C : row * a.C, a.u ? a.r_u[row] : 0.0f};
            const float r_y = a.r_y[row];
            const bool fresh = taken == 0 && row == r0;  // (nothing in the slice yet)
            float s1 = 0, s2 = 0;
            double s = 0;
            if (a.dh) {
                for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
                    const auto v = r.take(c, true);
                    float e[ANY], m[ANY];
#pragma unroll
                    for (int k = 0; k < ANY; ++k) e[k] = v.dh[k] * v.pre[k], m[k] = v.y[k] * r_y;
                    s += r.dot(e, m, c);
                }
                s1 = team.sum((float)s) * a.inv_c;
                s = 0;
            }
            for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
                const auto v = r.take(c, true);
                float post[ANY], pre[ANY], gate[ANY];  // the sums so far
#pragma unroll
                for (int k = 0; k < ANY; ++k) {
                    const int at = r.column(c, k);
                    post[k] = dpost && !fresh ? dpost[at] : 0.0f, pre[k] = dpre && !fresh ? dpre[at] : 0.0f, gate[k] = dgate && row > r0 ? dgate[at] : 0.0f;
                }
                float among = 0;
#pragma unroll
                for (int k = 0; k < ANY; ++k) {
                    const int at = c + 1024 * k;
                    if (at >= a.C) break;
                    const float d = r.through(v, k, r_y, s1), db = d * v.open[k];
                    if (dpre) dpre[at] = pre[k] + v.dh[k] * (v.y[k] * r_y);
                    if (a.dx) ((T *)a.dx)[r.base + at] = (T)d;
                    if (!a.u) continue;
                    if (dpost) dpost[at] = post[k] + db * v.n[k] * a.scale;
                    among += db * v.post[k] * v.n[k];
                    if (a.dgate) {
                        float dg = d * (v.n[k] * v.post[k]);
                        if (a.act) dg *= v.open[k] * (1.0f - v.open[k]);
                        if (dgate) dgate[at] = gate[k] + dg;
                        else ((T *)a.dgate)[r.base + at] = (T)dg;
                    }
                }
                s += among;
            }
            if (!a.du) continue;
            s2 = team.sum((float)s) * a.inv_c;
            for (int c = threadIdx.x; c < a.C; c += 1024 * ANY) {
                const auto v = r.take(c, true);
#pragma unroll
                for (int k = 0; k < ANY; ++k)
                    if (c + 1024 * k < a.C) ((T *)a.du)[r.base + c + 1024 * k] = (T)(r.r_u * (r.through(v, k, r_y, s1) * v.open[k] * v.post[k] - v.n[k] * s2));
            }
        }
        ++taken;
    }
}

// out[b][c] = sum over n of in[b][n][c] (columns 0 .. split - 1 to `out`, the others to `more`; either may be null) for columns from `first` on, 16 columns and 64 runs of rows a workgroup, joined in fp64
template <typename T>
__global__ __launch_bounds__(1024) void residual_join(const float *__restrict__ in, int64_t n, int columns, int split, T *__restrict__ out, T *__restrict__ more, int first) {
    __shared__ double sums[64][17];
    const int c = first + blockIdx.x * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
    const float *from = in + (int64_t)blockIdx.y * n * columns + min(c, columns - 1);
    double s = 0;
    for (int64_t k = run; k < n; k += 64 * 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + 64 * j < n ? from[(k + 64 * j) * columns] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    sums[run][threadIdx.x & 15] = s;
    __syncthreads();
    if (run == 0 && c < columns) {
        s = 0;
#pragma unroll 8
        for (int r = 0; r < 64; ++r) s += sums[r][threadIdx.x & 15];
        T *to = c < split ? out : more;
        if (to) to[(int64_t)blockIdx.y * split + (c < split ? c : c - split)] = (T)(float)s;
    }
}

// the same for few rows, a thread for each column (32 x 4096 columns of 16 rows: 29 us by runs of rows, 5 us so)
template <typename T>
__global__ __launch_bounds__(256) void residual_join_few(const float *__restrict__ in, int n, int columns, T *__restrict__ out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= columns) return;
    const float *from = in + (int64_t)blockIdx.y * n * columns + c;
    double s = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) s += from[(int64_t)k * columns];
    out[(int64_t)blockIdx.y * columns + c] = (T)(float)s;
}

namespace {

int check_residual(const char *what, int64_t rows, int64_t P, int64_t C, float scale, float eps, int act, int type) {
    if (rows < 0 || P < 1 || C < 1 || !(eps >= 0) || scale != scale || rows % P) return fail(HGQ_ERR_ARG, "%s: rows %lld (%lld a gate), channels %lld, epsilon %g, scale %g", what, (long long)rows, (long long)P, (long long)C, eps, scale);
    if (type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16 || act < 0 || act > 1) return fail(HGQ_ERR_ARG, "%s: unknown type or activation", what);
    if (C > 1 << 28 || rows > (int64_t)1 << 40) return fail(HGQ_ERR_UNSUPPORTED, "%s: %lld rows of %lld channels", what, (long long)rows, (long long)C);
    return HGQ_OK;
}

constexpr int RES_TERMS = 64;  // rows that a thread adds up one after the other, at most

struct ResidualPlan {
    int tpr, threads, grid, run;
    int64_t units, per_unit, cuts, slices;
};

// by_sample: a unit has rows of one sample, whose gate's gradient it adds up
ResidualPlan residual_plan(int64_t rows, int64_t P, int C, bool by_sample, bool gated) {
    ResidualPlan p;
    p.tpr = 1;
    while (p.tpr * RES_HELD < C && p.tpr < 64) p.tpr *= 2;
    if (p.tpr * RES_HELD < C) p.tpr = C > RES_WIDEST ? 1024 : (C + 64 * RES_HELD - 1) / (64 * RES_HELD) * 64;
    p.threads = p.tpr > 64 ? p.tpr : 256;
    const int teams = p.tpr > 64 ? 1 : 256 / p.tpr;
    // Workgroups of the backward pass.  Of two wavefronts: five a compute unit, as are resident (32768 x 768 bfloat16: 512 116 us, 1280 74, 2048 74).  Of three and
    // four: two, three with a gate, fewer than are resident (with four a compute unit 32768 x 1536 bfloat16 takes 139 instead of 134 us, 16384 x 1536 float32 133 and 131, 32768 x 2048
    // bfloat16 gated 249 and 240).  Of five to eight two, of more one (32768 x 4096: two 328, four 340).  Where wavefronts hold rows by themselves the same: each has a slice to join (131072 x
    // 64 float32: two 39, four 43, eight 48; 45930 x 333 float16 gated, read anew: two 66, three 62, four 67).
    const int64_t most = 256 * (p.threads > 512 ? 1 : p.threads > 256 ? 2 : p.threads == 128 ? 5 : gated ? 3 : 2);
    if (by_sample) {
        const int64_t samples = rows / P;
        p.cuts = samples < most ? (most + samples - 1) / samples : 1;
        const int64_t fewest = 2 * teams;  // rows that pay for a slice
        if (p.cuts > (P + fewest - 1) / fewest) p.cuts = (P + fewest - 1) / fewest;
        p.per_unit = std::min<int64_t>((P + p.cuts - 1) / p.cuts, RES_TERMS * teams);
        p.cuts = (P + p.per_unit - 1) / p.per_unit;
        p.units = samples * p.cuts;
    } else {
        p.per_unit = (rows + most - 1) / most;
        p.per_unit = std::min<int64_t>((p.per_unit + teams - 1) / teams * teams, RES_TERMS * teams);
        p.cuts = p.units = (rows + p.per_unit - 1) / p.per_unit;
    }
    p.grid = (int)(p.units < most ? p.units : most);
    // (of many rows a workgroup leaves several slices: what a thread adds up does not grow with the rows.  A slice takes as much as two rows in fp32, for 64 or more of them.)
    p.run = (int)(RES_TERMS / ((p.per_unit + teams - 1) / teams));
    const int64_t turns = (p.units + p.grid - 1) / p.grid, runs = (turns + p.run - 1) / p.run, before = (runs - 1) * p.grid;
    p.slices = before + std::min<int64_t>(p.grid, p.units - before * p.run);
    return p;
}

template <typename T, int KIND>
auto residual_fwd_of(const ResidualPlan &p, int C) {
    constexpr int N = Vec<T>::N;
    if (C < N) return residual_fwd<T, KIND, 256, TINY_ROWS>;
    if (p.tpr <= 64) return p.tpr == 64 ? residual_fwd<T, KIND, 256, WAVE_ROWS> : residual_fwd<T, KIND, 256, ROWS>;
    return p.tpr <= 512 ? residual_fwd<T, KIND, 512, ROWS> : residual_fwd<T, KIND, 1024, ROWS>;
}

template <typename T, int KIND>
auto residual_bwd_of(const ResidualPlan &p, int C) {
    constexpr int N = Vec<T>::N;
    if (C < N) return residual_bwd<T, KIND, 256, TINY_ROWS>;
    if (p.tpr <= 64) return p.tpr == 64 ? residual_bwd<T, KIND, 256, WAVE_ROWS> : residual_bwd<T, KIND, 256, ROWS>;
    return p.tpr <= 512 ? residual_bwd<T, KIND, 512, ROWS> : residual_bwd<T, KIND, 1024, ROWS>;
}

template <typename T, int KIND>
int forward(ResidualRows a, const ResidualPlan &p, hipStream_t st) {
    const bool wide = p.tpr > 64;
    const int teams = wide ? 1 : 256 / p.tpr;
    // threads a compute unit, all of them resident: five workgroups of 256 where wavefronts hold rows by themselves (1531 x 30 x 333 float16 with a gate, read anew: 40 us, four
    // 43, eight 44), 1024 where workgroups do (32768 x 4096 bfloat16 with a gate for samples 213 us, 1280 238, 2048 215; 8192 x 8192 102, 138, 107)
    const int64_t most = 256 * (wide ? 1024 : 1280) / p.threads, blocks = (a.rows + teams - 1) / teams, turns = (blocks + most - 1) / most, grid = (blocks + turns - 1) / turns, step = grid * teams;
    a.step_samples = step / a.P, a.step_rows = step % a.P;
    if (a.C > RES_WIDEST) hipLaunchKernelGGL((residual_fwd_any<T>), dim3((unsigned)grid), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((residual_fwd_of<T, KIND>(p, a.C)), dim3((unsigned)grid), dim3(p.threads), 0, st, a);
    return check_launch("hgq_residual_norm_fwd");
}

template <typename T>
int join(const float *in, int64_t n, unsigned many, int columns, int split, T *out, T *more, hipStream_t st) {
    constexpr int most = 1 << 25;  // columns of a launch (one of 2^32 threads or more runs some of them, and says nothing)
    int rc = HGQ_OK;
    for (int first = 0; first < columns && !rc; first += most) {
        const int left = columns - first, here = left < most ? left : most;
        hipLaunchKernelGGL(residual_join<T>, dim3((unsigned)((here + 15) / 16), many), dim3(1024), 0, st, in, n, columns, split, out, more, first);
        rc = check_launch("hgq_residual_norm_bwd");
    }
    return rc;
}

template <typename T, int KIND>
int backward(const ResidualRows &a, const ResidualPlan &p, float *dpost, float *dpre, hipStream_t st) {
    const char *what = "hgq_residual_norm_bwd";
    if (a.C > RES_WIDEST) hipLaunchKernelGGL((residual_bwd_any<T>), dim3(p.grid), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((residual_bwd_of<T, KIND>(p, a.C)), dim3(p.grid), dim3(p.threads), 0, st, a);
    int rc = check_launch(what);
    if (!rc && a.slices) {
        rc = join(a.slices, p.slices, 1, 2 * a.C, a.C, dpost, dpre, st);
    }
    if (!rc && a.gate_slices) {
        const int64_t samples = a.rows / a.P;
        for (int64_t b = 0; b < samples && !rc; b += 65535) {
            const unsigned many = (unsigned)(samples - b < 65535 ? samples - b : 65535);
            const float *slices = a.gate_slices + b * p.cuts * a.C;
            T *dgate = (T *)a.dgate + b * a.C;
            if (p.cuts <= 64) hipLaunchKernelGGL(residual_join_few<T>, dim3((unsigned)((a.C + 255) / 256), many), dim3(256), 0, st, slices, (int)p.cuts, a.C, dgate);
            else rc = join(slices, p.cuts, many, a.C, a.C, dgate, (T *)nullptr, st);
            if (!rc) rc = check_launch(what);
        }
    }
    return rc;
}

bool slices_of_gate(const ResidualPlan &p, int C) { return p.cuts > 1 || C > RES_WIDEST; }

template <typename T>
auto forward_of(int kind) {
    return kind == NO_UPDATE ? forward<T, NO_UPDATE> : kind == NO_GATE ? forward<T, NO_GATE> : kind == GATED ? forward<T, GATED> : forward<T, GATED_SAMPLES>;
}

template <typename T>
auto backward_of(int kind) {
    return kind == NO_UPDATE ? backward<T, NO_UPDATE> : kind == NO_GATE ? backward<T, NO_GATE> : kind == GATED ? backward<T, GATED> : backward<T, GATED_SAMPLES>;
}

}  // namespace
}  // namespace hgq

using namespace hgq;

extern "C" int hgq_residual_norm_fwd(const void *x, const void *u, const void *gate, const float *post, const float *pre, void *y, void *h, float *r_u, float *r_y,
                                     int64_t rows, int64_t P, int64_t C, float scale, float eps, int act, int type, void *stream) {
    const char *what = "hgq_residual_norm_fwd";
    int rc = check_residual(what, rows, P, C, scale, eps, act, type);
    if (rc || rows == 0) return rc;
    if (!x || !h || (u && !y) || (gate && !u)) return fail(HGQ_ERR_ARG, "%s: null pointer", what);
    if (!gate) P = 1;
    ResidualRows a = {};
    a.x = x, a.u = u, a.gate = gate, a.post = post, a.pre = pre, a.y = y, a.h = h, a.r_u = u ? r_u : nullptr, a.r_y = r_y;
    const ResidualPlan p = residual_plan(rows, P, (int)C, false, false);
    a.rows = rows, a.P = P, a.C = (int)C, a.tpr = p.tpr, a.act = act, a.by_sample = P > 1, a.samples = rows / P, a.scale = scale, a.eps = eps, a.inv_c = (float)(1.0 / (double)C);
    const int kind = !u ? NO_UPDATE : !gate ? NO_GATE : P > 1 ? GATED_SAMPLES : GATED;
    return (type == HGQ_TYPE_F32 ? forward_of<float>(kind) : type == HGQ_TYPE_BF16 ? forward_of<__bf16>(kind) : forward_of<_Float16>(kind))(a, p, (hipStream_t)stream);
}

extern "C" int64_t hgq_residual_norm_bwd_workspace(int64_t rows, int64_t P, int64_t C, int type) {
    if (check_residual("hgq_residual_norm_bwd_workspace", rows, P, C, 1.0f, 0.0f, 0, type)) return -1;
    if (rows == 0) return 0;
    int64_t most = 0;
    for (int kind = 0; kind < 3; ++kind) {  // no gate, one like x, one for a sample's rows
        const bool by_sample = kind == 2 && P > 1;
        const ResidualPlan p = residual_plan(rows, P, (int)C, by_sample, kind > 0);
        const int64_t floats = 2 * p.slices * C + (by_sample && slices_of_gate(p, (int)C) ? p.units * C : 0);
        most = floats > most ? floats : most;
    }
    return most;
}

extern "C" int hgq_residual_norm_bwd(const void *dy, const void *dh, const void *x, const void *u, const void *gate, const float *post, const float *pre,
                                     const float *r_u, const float *r_y, void *dx, void *du, void *dgate, float *dpost, float *dpre, float *workspace,
                                     int64_t rows, int64_t P, int64_t C, float scale, float eps, int act, int type, void *stream) {
    const char *what = "hgq_residual_norm_bwd";
    int rc = check_residual(what, rows, P, C, scale, eps, act, type);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {
        if (dpost && (rc = fill_f32(dpost, 0.0f, C, st))) return rc;
        return dpre ? fill_f32(dpre, 0.0f, C, st) : HGQ_OK;
    }
    if (!x || !r_y || (u && !r_u) || (!dy && !dh) || !workspace || (gate && !u) || (dgate && !gate) || (!u && (du || dpost))) return fail(HGQ_ERR_ARG, "%s: null pointer", what);
    if (!gate) P = 1;
    const ResidualPlan p = residual_plan(rows, P, (int)C, P > 1, gate != nullptr);
    ResidualRows a = {};
    a.x = x, a.u = u, a.gate = gate, a.dy = dy, a.dh = dh, a.post = post, a.pre = pre, a.dx = dx, a.du = du, a.dgate = dgate;
    a.r_u = (float *)r_u, a.r_y = (float *)r_y, a.slices = dpost || dpre ? workspace : nullptr;
    a.gate_slices = dgate && P > 1 && slices_of_gate(p, (int)C) ? workspace + 2 * p.slices * C : nullptr;
    a.rows = rows, a.P = P > 1 ? P : rows, a.units = p.units, a.per_unit = p.per_unit, a.cuts = p.cuts, a.run = p.run;
    a.C = (int)C, a.tpr = p.tpr, a.act = act, a.by_sample = P > 1, a.samples = rows / P, a.scale = scale, a.eps = eps, a.inv_c = (float)(1.0 / (double)C);
    const int kind = !u ? NO_UPDATE : !gate ? NO_GATE : P > 1 ? GATED_SAMPLES : GATED;
    return (type == HGQ_TYPE_F32 ? backward_of<float>(kind) : type == HGQ_TYPE_BF16 ? backward_of<__bf16>(kind) : backward_of<_Float16>(kind))(a, p, dpost, dpre, st);
}
