// AdamW over many variables in one launch, with both moments in 32 bits or in 8 bits, and the global norm of their gradients.
//
// A step t = 1, 2, ... with a variable's gradient g (the pieces `g`, `side[s] * side_scale[s]` and the constant l1 added up):
//     g <- g * c,  c = 1 or clipnorm / norm over all variables
//     m <- m + (g - m) (1 - beta_1)          v <- v + (g g - v) (1 - beta_2)          r = sqrt(v)
//     w <- clip(w - w (lr decay) - m alpha / (r + epsilon), lo, hi),   alpha = lr sqrt(1 - beta_2^t) / (1 - beta_1^t)
// in fp32 whatever the type of w and g; w is rounded to its type once, at the end.
//
// Moments in 8 bits.  m and r (not v: the square root halves the exponents a block spans) are E4M3 codes times a power of two
// 2^(s - 127) per 256 elements, s = max(exponent field of the block's largest magnitude - 7, 1), so the largest lies in [128, 256).
// The step of a slow average is far below half a code (1 - beta_2 = 0.001 against code distances of 1/16 to 1/8), so rounding
// to the nearest code would never move it: codes are rounded stochastically, which keeps the average unbiased.  The 16-bit numbers
// come from Philox4x32-7 (seven rounds: the fewest that pass the statistical tests of Salmon et al., SC'11; the rounding
// draws 32 bits per element): word e % 4 of counter (e / 4, t), low half for m and high half for r.  As fp32 numbers scaled by
// 2^-120, E4M3 values have their code, normal and subnormal, in bits 20 to 27, so rounding is one addition to the bits below and a shift.
// An r above zero keeps at least the smallest code: a zero would let epsilon alone divide the next step.
#include <math.h>

#include "hgq_device.h"
#include "hgq_host.h"

namespace hgq {

constexpr int ADAMW_ITEMS = 28, ADAMW_PIECES = 32;
// A step that touches more than the card's 256 MB cache passes through it once: accesses that leave no trace there, four blocks per
// wavefront in flight, a workgroup per 4096 elements.  150 million elements, 4.2 GB: 851 -> 720 us (5.9 TB/s; the card copies at 5.0), with
// moments in 8 bits, 2.4 GB: 552 -> 437 us (now 401 - 415, its 88 vector instructions per element close behind); 37 million bfloat16: 164 ->
// 137 us.  A smaller step leaves its weights for the next forward pass; two blocks, and up to 2048 workgroups that go over 2048
// elements at a time (4 million elements: 22 us either way).
constexpr int64_t ADAMW_CACHE = (int64_t)256 << 20;
constexpr int ADAMW_CHUNK = 2048, ADAMW_STREAM_CHUNK = 4096;  // elements a workgroup takes at a time, in blocks of 256
constexpr int ADAMW_GRID = 2048;
// Gradients are read around the cache whatever their size: 150 million 145 -> 89 us (6.7 TB/s), 24 million 24 -> 21 us, and the update that
// follows takes as long to within 3 %.
constexpr int NORM_LOADS = 8, NORM_GRID = 1024;

struct AdamwItem {
    void *w;
    const void *g;
    void *m, *v;
    uint8_t *m_scale, *v_scale;
    int64_t n, first;
    float l1, lo, hi, decay;
    char type, vec;       // vec: a plain gradient and aligned memory, four elements per access
    char bounded;         // lo or hi is finite
    short piece, pieces;  // its entries of the launch's list of further gradient pieces
};
struct AdamwLaunch {
    AdamwItem item[ADAMW_ITEMS];
    const float *side[ADAMW_PIECES], *side_scale[ADAMW_PIECES];
    uint32_t start[ADAMW_ITEMS + 1];  // first chunk of each item, then their number in all further entries
};
struct AdamwSum {
    const float *term[HGQ_SUM_BATCH];
    int n;
    float *out;
};

// The item of a chunk: comparisons with all starts, not one load after the other.  A step of 28 variables with 13 thousand elements: 6.5 ->
// 5.4 us; 150 million elements past the cache 730 -> 722 us.
__device__ __forceinline__ int item_of(const AdamwLaunch &a, uint32_t chunk) {
    int i = 0;
#pragma unroll
    for (int k = 1; k < ADAMW_ITEMS; ++k) i += chunk >= a.start[k];
    return i;
}

__device__ __forceinline__ float load_as_f32(const void *p, int64_t e, int type) {
    if (type == HGQ_TYPE_F32) return ((const float *)p)[e];
    const uint16_t h = ((const uint16_t *)p)[e];
    if (type == HGQ_TYPE_BF16) return __uint_as_float((uint32_t)h << 16);
    _Float16 f;
    __builtin_memcpy(&f, &h, 2);
    return (float)f;
}

__device__ __forceinline__ void store_f32_as(void *p, int64_t e, int type, float v) {
    if (type == HGQ_TYPE_F32) {
        ((float *)p)[e] = v;
    } else if (type == HGQ_TYPE_BF16) {  // to the nearest, ties to even; a NaN stays one
        const uint32_t b = __float_as_uint(v);
        ((uint16_t *)p)[e] = v != v ? (uint16_t)((b >> 16) | 0x40) : (uint16_t)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
    } else {
        ((_Float16 *)p)[e] = (_Float16)v;
    }
}

// the gradient of element e: its pieces in the order of the descriptor, then the regularizer's constant
__device__ __forceinline__ float gradient(const AdamwLaunch &a, const AdamwItem &it, int64_t e) {
    float g = it.g ? load_as_f32(it.g, e, it.type) : 0.0f;
    for (int s = 0; s < it.pieces; ++s) {
        const float *scale = a.side_scale[it.piece + s], d = a.side[it.piece + s][e];
        g = __fadd_rn(g, scale ? __fmul_rn(scale[0], d) : d);
    }
    return __fadd_rn(g, it.l1);
}

__device__ __forceinline__ void philox4x32_7(uint64_t counter, uint64_t step, uint64_t seed, uint32_t (&out)[4]) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, c1 = (uint32_t)p1, c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1, c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// E4M3 code of a finite magnitude under the block's scale byte s, rounded by the 16-bit number h
__device__ __forceinline__ uint32_t e4m3_code(float a, int s, uint32_t h) { return (__float_as_uint(ldexpf(a, 7 - s)) + (h << 4)) >> 20; }

template <int J>
__device__ __forceinline__ float e4m3_value(uint32_t codes, int s) {  // of byte J
    return ldexpf(__builtin_amdgcn_cvt_f32_fp8((int)codes, J), s - 127);
}

__device__ __forceinline__ uint32_t exponent_field(float v) {  // of finite magnitudes; the others do not count
    const uint32_t e = (__float_as_uint(v) >> 23) & 0xff;
    return e == 255 ? 0 : e;
}

struct AdamwStep {
    float c, alpha, lr, one_minus_b1, one_minus_b2, eps;
    uint64_t t, seed;
};

// w <- the updated weight; m and r already hold the new moments.  The quotient is a product with the hardware's reciprocal (one unit in
// the last place; r + eps lies in [2^-75, 2^65] or is zero): the step is far smaller than w, and a rounded division takes ten instructions.
__device__ __forceinline__ float adamw_weight(float w, float m, float r, const AdamwItem &it, const AdamwStep &k) {
    w = __fsub_rn(w, __fmul_rn(w, __fmul_rn(k.lr, it.decay)));
    return __fsub_rn(w, __fmul_rn(__fmul_rn(m, k.alpha), __builtin_amdgcn_rcpf(__fadd_rn(r, k.eps))));
}

__device__ __forceinline__ float adamw_clip(float w, const AdamwItem &it) {
    return w < it.lo ? it.lo : w > it.hi ? it.hi : w;  // (not a number stays that)
}

// the new moments of one element with gradient g: m, v and r = sqrt(v)
__device__ __forceinline__ void adamw_moments(float g, float &m, float &v, float &r, const AdamwStep &k) {
    g = __fmul_rn(g, k.c);
    m = __fadd_rn(m, __fmul_rn(__fsub_rn(g, m), k.one_minus_b1));
    v = __fadd_rn(v, __fmul_rn(__fsub_rn(__fmul_rn(g, g), v), k.one_minus_b2));
    // The rounded root: __fsqrt_rn is the hardware's here, a unit in the last place off, which moves a code where r lies on a border of its
    // rounding (150 million elements: 17 codes of r).  Nine vector instructions more: with 8-bit moments 401 -> 415 us there, 821 -> 823 with 32-bit ones.
    r = sqrtf(v);
}

typedef uint16_t halves_t __attribute__((ext_vector_type(2)));

// Codes of a wavefront's block, four neighbours per lane (those behind the last element: zeros): m and r go in, the scale bytes
// and a word of four codes each come out.
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&r)[4], uint64_t element, const AdamwStep &k, int &sm, int &sr,
                                             uint32_t &cm, uint32_t &cr) {
    // magnitudes by their bits: in the order of the numbers, infinities and what is not a number behind them
    uint32_t mm = 0, rm = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mm = max(mm, __float_as_uint(m[j]) & 0x7fffffffu), rm = max(rm, __float_as_uint(r[j]));
    const bool plain = __all(max(mm, rm) < 0x7f800000u);
    uint32_t both = mm >> 23 << 16 | rm >> 23;  // both exponent fields in the halves of one word: one exchange for the two maxima
    if (!plain) {                               // what is not finite does not count
        uint32_t em = 0, er = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) em = max(em, exponent_field(m[j])), er = max(er, exponent_field(r[j]));
        both = em << 16 | er;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint32_t other = (uint32_t)__shfl_xor((int)both, d);
        halves_t a, b;
        __builtin_memcpy(&a, &both, 4), __builtin_memcpy(&b, &other, 4);
        a = __builtin_elementwise_max(a, b);
        __builtin_memcpy(&both, &a, 4);
    }
    sm = max((int)(both >> 16), 8) - 7, sr = max((int)(both & 0xffff), 8) - 7;
    uint32_t h[4];
    philox4x32_7(element >> 2, k.t, k.seed, h);
    cm = cr = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t a = e4m3_code(fabsf(m[j]), sm, h[j] & 0xffff), b = e4m3_code(r[j], sr, h[j] >> 16);
        b = max(b, min(__float_as_uint(r[j]), 1u));  // (above zero: the smallest code at least)
        if (!plain) {
            if (exponent_field(m[j]) == 0 && !(fabsf(m[j]) < 1.0f)) a = 0x7f;
            if (exponent_field(r[j]) == 0 && !(r[j] < 1.0f)) b = 0x7f;
        }
        cm |= (a | ((__float_as_uint(m[j]) >> 24) & 0x80u)) << (8 * j), cr |= b << (8 * j);
    }
}

// a wavefront's block of 256 elements at b, element by element: any alignment, any gradient pieces, any end
template <int BITS>
__device__ __forceinline__ void adamw_block_any(const AdamwLaunch &a, const AdamwItem &it, const AdamwStep &k, int64_t b) {
    const int lane = threadIdx.x & 63;
    const int64_t e = b + lane * 4;
    float m[4], v[4], r[4], g[4], w[4];
    int sm = 0, sr = 0;
    if (BITS == 8) sm = it.m_scale[b >> 8], sr = it.v_scale[b >> 8];
    // (all loads before the first store: the compiler cannot know that the arrays do not overlap)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = v[j] = r[j] = g[j] = w[j] = 0.0f;
        if (e + j < it.n) {
            g[j] = gradient(a, it, e + j), w[j] = load_as_f32(it.w, e + j, it.type);
            if (BITS == 8) {
                m[j] = e4m3_value<0>(((const uint8_t *)it.m)[e + j], sm), v[j] = e4m3_value<0>(((const uint8_t *)it.v)[e + j], sr);
                v[j] = __fmul_rn(v[j], v[j]);
            } else {
                m[j] = ((const float *)it.m)[e + j], v[j] = ((const float *)it.v)[e + j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (e + j < it.n) {
            adamw_moments(g[j], m[j], v[j], r[j], k);
            store_f32_as(it.w, e + j, it.type, adamw_clip(adamw_weight(w[j], m[j], r[j], it, k), it));
            if (BITS == 32) ((float *)it.m)[e + j] = m[j], ((float *)it.v)[e + j] = v[j];
        }
    if (BITS == 8) {
        uint32_t cm, cr;
        encode_block(m, r, (uint64_t)(it.first + e), k, sm, sr, cm, cr);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e + j < it.n) ((uint8_t *)it.m)[e + j] = (uint8_t)(cm >> (8 * j)), ((uint8_t *)it.v)[e + j] = (uint8_t)(cr >> (8 * j));
        if (lane == 0) it.m_scale[b >> 8] = (uint8_t)sm, it.v_scale[b >> 8] = (uint8_t)sr;
    }
}

typedef uint32_t words2_t __attribute__((ext_vector_type(2)));
typedef float floats4_t __attribute__((ext_vector_type(4)));

// four neighbours of an aligned array as they lie in memory
template <typename T>
struct Four;
template <>
struct Four<float> {
    typedef floats4_t raw;
};
template <>
struct Four<__bf16> {
    typedef __bf16 raw __attribute__((ext_vector_type(4)));
};
template <>
struct Four<_Float16> {
    typedef _Float16 raw __attribute__((ext_vector_type(4)));
};

template <bool STREAM, typename V>
__device__ __forceinline__ V read(const void *p) {
    return STREAM ? __builtin_nontemporal_load((const V *)p) : *(const V *)p;
}

template <bool STREAM, typename V>
__device__ __forceinline__ void write(void *p, V v) {
    if (STREAM) __builtin_nontemporal_store(v, (V *)p);
    else *(V *)p = v;
}

// N of a wavefront's whole blocks, at b and every 1024 elements on: four elements per access, all loads before the first use
template <int BITS, typename T, int N, bool STREAM>
__device__ __forceinline__ void adamw_blocks(const AdamwItem &it, const AdamwStep &k, int64_t b) {
    typedef typename Four<T>::raw raw;
    const int lane = threadIdx.x & 63;
    const int64_t e = b + lane * 4;
    raw w[N], g[N];
    floats4_t m[N], v[N];
    uint32_t cm[N], cr[N];
    int sm[N], sr[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        g[n] = read<STREAM, raw>((const T *)it.g + e + 1024 * n);
        w[n] = read<STREAM, raw>((const T *)it.w + e + 1024 * n);
        if (BITS == 32) {
            m[n] = read<STREAM, floats4_t>((const float *)it.m + e + 1024 * n), v[n] = read<STREAM, floats4_t>((const float *)it.v + e + 1024 * n);
        } else {
            cm[n] = read<STREAM, uint32_t>((const uint8_t *)it.m + e + 1024 * n), cr[n] = read<STREAM, uint32_t>((const uint8_t *)it.v + e + 1024 * n);
            sm[n] = it.m_scale[(b >> 8) + 4 * n], sr[n] = it.v_scale[(b >> 8) + 4 * n];
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float mm[4], vv[4], rr[4], ww[4];
        if (BITS == 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) mm[j] = m[n][j], vv[j] = v[n][j];
        } else {
            mm[0] = e4m3_value<0>(cm[n], sm[n]), mm[1] = e4m3_value<1>(cm[n], sm[n]), mm[2] = e4m3_value<2>(cm[n], sm[n]), mm[3] = e4m3_value<3>(cm[n], sm[n]);
            vv[0] = e4m3_value<0>(cr[n], sr[n]), vv[1] = e4m3_value<1>(cr[n], sr[n]), vv[2] = e4m3_value<2>(cr[n], sr[n]), vv[3] = e4m3_value<3>(cr[n], sr[n]);
#pragma unroll
            for (int j = 0; j < 4; ++j) vv[j] = __fmul_rn(vv[j], vv[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            adamw_moments(__fadd_rn((float)g[n][j], it.l1), mm[j], vv[j], rr[j], k);
            ww[j] = adamw_weight((float)w[n][j], mm[j], rr[j], it, k);
            m[n][j] = mm[j], v[n][j] = vv[j];
        }
        if (it.bounded)
#pragma unroll
            for (int j = 0; j < 4; ++j) ww[j] = adamw_clip(ww[j], it);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[n][j] = (T)ww[j];
        write<STREAM>((T *)it.w + e + 1024 * n, w[n]);
        if (BITS == 32) {
            write<STREAM>((float *)it.m + e + 1024 * n, m[n]), write<STREAM>((float *)it.v + e + 1024 * n, v[n]);
        } else {
            encode_block(mm, rr, (uint64_t)(it.first + e + 1024 * n), k, sm[n], sr[n], cm[n], cr[n]);
            write<STREAM>((uint8_t *)it.m + e + 1024 * n, cm[n]), write<STREAM>((uint8_t *)it.v + e + 1024 * n, cr[n]);
            if (lane == 0) it.m_scale[(b >> 8) + 4 * n] = (uint8_t)sm[n], it.v_scale[(b >> 8) + 4 * n] = (uint8_t)sr[n];
        }
    }
}

// one variable's elements [e0, e0 + a chunk): a lane takes four neighbours, a wavefront 256 - the block that shares a scale
template <int BITS, bool STREAM>
__device__ __forceinline__ void adamw_chunk(const AdamwLaunch &a, const AdamwItem &it, const AdamwStep &k, int64_t e0) {
    constexpr int CHUNK = STREAM ? ADAMW_STREAM_CHUNK : ADAMW_CHUNK, N = CHUNK / 1024;
    const int64_t b0 = e0 + (threadIdx.x >> 6) * 256;
    if (it.vec && e0 + CHUNK <= it.n) {
        if (it.type == HGQ_TYPE_F32) adamw_blocks<BITS, float, N, STREAM>(it, k, b0);
        else if (it.type == HGQ_TYPE_BF16) adamw_blocks<BITS, __bf16, N, STREAM>(it, k, b0);
        else adamw_blocks<BITS, _Float16, N, STREAM>(it, k, b0);
        return;
    }
    for (int64_t b = b0; b < e0 + CHUNK && b < it.n; b += 1024) {
        if (it.vec && it.type == HGQ_TYPE_F32 && b + 256 <= it.n) adamw_blocks<BITS, float, 1, STREAM>(it, k, b);
        else adamw_block_any<BITS>(a, it, k, b);
    }
}

// sum of the workgroup's values, in a fixed order, returned to every thread
__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) v += lds[w];
    __syncthreads();
    return v;
}

// The step's number, the powers of the decay rates and the learning rate live in device memory (hgq_adamw_state), so a recorded launch
// moves on at every replay.  All workgroups read them; in a step's last launch each then takes a ticket, and the one with the last
// ticket writes the next step's.  Tickets of one counter come one every 27 ns (2048 workgroups: 55 us, more than an update of 4 million
// elements takes), so there are 32 counters in cache lines of their own, and one for those that finish them; and a workgroup takes
// its ticket when it begins, so that the answer is there when it ends.
template <int BITS, bool STREAM>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwLaunch a, AdamwSum sum, hgq_adamw_state *state, double b1, double b2, float eps,
                                                    float clipnorm, const double *parts, int n_parts, const float *joined, float *norm_out, uint64_t seed,
                                                    int last) {
    __shared__ double lds[4];
    if (sum.n > 0 && blockIdx.x == 0 && threadIdx.x == 0) {  // the step's loss terms, which the update does not read
        float v = sum.term[0][0];
        for (int t = 1; t < sum.n; ++t) v = __fadd_rn(v, sum.term[t][0]);
        sum.out[0] = v;
    }
    // What the memory has to answer first - the state, the parts of the norm, the descriptor of the first chunk - is asked for at once, and only then
    // waited for (0.88 million elements: 8.1 -> 7.6 us).
    const double lr = state->lr, power_1 = state->beta_1_power, power_2 = state->beta_2_power;
    const int64_t steps = state->step;
    double squares = 0;
    if (n_parts > 0 && !joined)
        for (int p = threadIdx.x; p < n_parts; p += 256) squares += parts[p];
    const int first = item_of(a, blockIdx.x);
    __shared__ AdamwStep shared;
    uint32_t left = 1;  // tickets not taken before this workgroup's, of its counter
    int64_t t = 0;
    double p1 = 0, p2 = 0;
    const uint32_t counter = gridDim.x > HGQ_ADAMW_TICKETS ? 1 + blockIdx.x % HGQ_ADAMW_TICKETS : HGQ_ADAMW_TICKETS + 1;
    if (threadIdx.x == 0) {
        t = steps + 1, p1 = power_1 * b1, p2 = power_2 * b2;
        shared.alpha = (float)(lr * sqrt(1.0 - p2) / (1.0 - p1)), shared.lr = (float)lr, shared.t = (uint64_t)t;
        asm volatile("" ::"v"(t), "v"(p1), "v"(p2), "v"(lr) : "memory");  // (the reads are done before the ticket is taken)
        if (last) {
            const uint32_t all = counter <= HGQ_ADAMW_TICKETS ? (gridDim.x - counter) / HGQ_ADAMW_TICKETS + 1 : gridDim.x;
            left = all - 1 - atomicAdd(&state->ticket[counter][0], 1u);
        }
    }
    __syncthreads();
    AdamwStep k = shared;
    k.seed = seed, k.one_minus_b1 = (float)(1.0 - b1), k.one_minus_b2 = (float)(1.0 - b2), k.eps = eps;
    k.c = 1.0f;
    if (n_parts > 0) {
        const float norm = joined ? joined[0] : (float)sqrt(block_sum(squares, lds));
        // No clipping up to the bound; a norm that is not finite makes every step not a number.  The product with the rounded reciprocal is
        // Keras' order of operations, a rounding more than the quotient, which stands in where the reciprocal is no normal number.
        const float inverse = __fdiv_rn(1.0f, norm);
        const bool normal = inverse >= 0x1p-126f && inverse < __builtin_inff();
        k.c = norm <= clipnorm ? 1.0f : !(norm < __builtin_inff()) ? __builtin_nanf("") : normal ? fminf(__fmul_rn(clipnorm, inverse), 1.0f) : __fdiv_rn(clipnorm, norm);
        if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
    }
    for (uint32_t c = blockIdx.x; c < a.start[ADAMW_ITEMS]; c += gridDim.x) {
        const int i = c == blockIdx.x ? first : item_of(a, c);
        adamw_chunk<BITS, STREAM>(a, a.item[i], k, (int64_t)(c - a.start[i]) * (STREAM ? ADAMW_STREAM_CHUNK : ADAMW_CHUNK));
    }
    if (left) return;
    state->ticket[counter][0] = 0;
    if (counter <= HGQ_ADAMW_TICKETS) {
        if (atomicAdd(&state->ticket[HGQ_ADAMW_TICKETS + 1][0], 1u) != HGQ_ADAMW_TICKETS - 1) return;
        state->ticket[HGQ_ADAMW_TICKETS + 1][0] = 0;
    }
    state->step = t, state->beta_1_power = p1, state->beta_2_power = p2;
}

// squares of four neighbours; (v ^ 2 of fp32 has 48 bits and stays exact in fp64)
template <typename T>
__device__ __forceinline__ double squares(const typename Four<T>::raw &g, float l1) {
    double v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double d = __fadd_rn((float)g[j], l1);
        v += d * d;
    }
    return v;
}

// one variable's elements [e0, e0 + NORM_LOADS * 1024), whole and aligned: all loads before the first use
template <typename T>
__device__ __forceinline__ double norm_chunk(const AdamwItem &it, int64_t e0) {
    typedef typename Four<T>::raw raw;
    raw g[NORM_LOADS];
#pragma unroll
    for (int n = 0; n < NORM_LOADS; ++n) g[n] = __builtin_nontemporal_load((const raw *)((const T *)it.g + e0 + 1024 * n + 4 * threadIdx.x));
    double v = 0;
#pragma unroll
    for (int n = 0; n < NORM_LOADS; ++n) v += squares<T>(g[n], it.l1);
    return v;
}

// sums of squares, one per workgroup: in fp64, so that no finite gradient overflows and their order does not show
__global__ __launch_bounds__(256) void norm_parts_kernel(AdamwLaunch a, int chunk, double *parts) {
    __shared__ double lds[4];
    double v = 0;
    int i = item_of(a, blockIdx.x);
    for (uint32_t c = blockIdx.x; c < a.start[ADAMW_ITEMS]; c += gridDim.x) {
        while (c >= a.start[i + 1]) ++i;
        const AdamwItem &it = a.item[i];
        const int64_t e0 = (int64_t)(c - a.start[i]) * chunk, end = e0 + chunk < it.n ? e0 + chunk : it.n;
        if (it.vec && end - e0 == NORM_LOADS * 1024) {
            v += it.type == HGQ_TYPE_F32 ? norm_chunk<float>(it, e0) : it.type == HGQ_TYPE_BF16 ? norm_chunk<__bf16>(it, e0) : norm_chunk<_Float16>(it, e0);
            continue;
        }
        for (int64_t e = e0 + threadIdx.x; e < end; e += 256) {
            const double g = gradient(a, it, e);
            v += g * g;
        }
    }
    v = block_sum(v, lds);
    if (threadIdx.x == 0) parts[blockIdx.x] = v;
}

__global__ __launch_bounds__(256) void norm_finish_kernel(const double *parts, int n, float *out) {
    __shared__ double lds[4];
    double v = 0;
    for (int p = threadIdx.x; p < n; p += 256) v += parts[p];
    v = block_sum(v, lds);
    if (threadIdx.x == 0) out[0] = (float)sqrt(v);
}

}  // namespace hgq

using namespace hgq;

namespace {

// Goes over `items` in launches of up to ADAMW_ITEMS variables and ADAMW_PIECES further gradient pieces: fn(launch, last).
// Descriptors travel as launch arguments (4 KB at most), so the calls are safe under HIP graph capture.
template <class F>
int for_launches(const hgq_adamw_item *items, int count, int chunk, F fn) {
    int at = 0;
    bool done = false;
    while (!done) {
        AdamwLaunch a = {};
        int n = 0, pieces = 0;
        uint64_t chunks = 0;
        for (; at < count && n < ADAMW_ITEMS; ++at) {
            const hgq_adamw_item &s = items[at];
            if (s.n == 0) continue;
            int own = 0;
            for (int k = 0; k < HGQ_SGD_SIDES; ++k) own += s.side[k] != nullptr;
            const uint64_t own_chunks = ((uint64_t)s.n + chunk - 1) / chunk;
            if (pieces + own > ADAMW_PIECES || (n > 0 && chunks + own_chunks > 0x7fffffffu)) break;
            AdamwItem &d = a.item[n];
            d.w = s.w, d.g = s.g, d.m = s.m, d.v = s.v, d.m_scale = s.m_scale, d.v_scale = s.v_scale, d.n = s.n, d.first = s.first;
            d.l1 = s.l1, d.lo = s.lo, d.hi = s.hi, d.decay = s.decay, d.type = (char)s.type, d.bounded = !(s.lo == -INFINITY && s.hi == INFINITY), d.piece = (short)pieces, d.pieces = (short)own;
            const uintptr_t size = s.type == HGQ_TYPE_F32 ? 4 : 2, moment = s.m_scale ? 1 : 4;
            d.vec = own == 0 && (((uintptr_t)s.w | (uintptr_t)s.g) & (4 * size - 1)) == 0 && (((uintptr_t)s.m | (uintptr_t)s.v) & (4 * moment - 1)) == 0;
            for (int k = 0; k < HGQ_SGD_SIDES; ++k)
                if (s.side[k]) a.side[pieces] = s.side[k], a.side_scale[pieces] = s.side_scale[k], ++pieces;
            a.start[n++] = (uint32_t)chunks;
            chunks += own_chunks;
        }
        for (int k = n; k <= ADAMW_ITEMS; ++k) a.start[k] = (uint32_t)chunks;
        while (at < count && items[at].n == 0) ++at;
        done = at >= count;
        const int rc = fn(a, done);
        if (rc) return rc;
    }
    return HGQ_OK;
}

int check_items(const char *what, const hgq_adamw_item *items, int count, int bits) {
    if (count < 0 || (count > 0 && !items)) return fail(HGQ_ERR_ARG, "%s: bad arguments", what);
    for (int t = 0; t < count; ++t) {
        const hgq_adamw_item &s = items[t];
        if (s.n < 0 || s.n > (int64_t)1 << 40) return fail(HGQ_ERR_ARG, "%s: bad number of elements in item %d", what, t);
        if (s.n == 0) continue;
        bool any = s.g != nullptr;
        for (int k = 0; k < HGQ_SGD_SIDES; ++k) any = any || s.side[k];
        if (!any || (bits && (!s.w || !s.m || !s.v))) return fail(HGQ_ERR_ARG, "%s: null pointer in item %d", what, t);
        if (s.type != HGQ_TYPE_F32 && s.type != HGQ_TYPE_BF16 && s.type != HGQ_TYPE_F16) return fail(HGQ_ERR_ARG, "%s: unknown type in item %d", what, t);
        if (bits == 8 && (!s.m_scale || !s.v_scale || s.first < 0 || s.first % HGQ_ADAMW_BLOCK))
            return fail(HGQ_ERR_ARG, "%s: item %d has no scales, or its first element is not a multiple of %d", what, t, HGQ_ADAMW_BLOCK);
    }
    return HGQ_OK;
}

int norm_grid(const AdamwLaunch &a) {
    const uint32_t chunks = a.start[ADAMW_ITEMS];
    return (int)(chunks < NORM_GRID ? chunks : NORM_GRID);
}

}  // namespace

extern "C" int64_t hgq_global_norm_parts(const hgq_adamw_item *items, int count) {
    if (check_items("hgq_global_norm_parts", items, count, 0)) return -1;
    int64_t parts = 0;
    const int chunk = NORM_LOADS * 1024;
    for_launches(items, count, chunk, [&](const AdamwLaunch &a, bool) {
        parts += norm_grid(a);
        return HGQ_OK;
    });
    return parts;
}

extern "C" int hgq_global_norm(const hgq_adamw_item *items, int count, double *parts, float *out, void *stream) {
    int rc = check_items("hgq_global_norm", items, count, 0);
    if (rc) return rc;
    int64_t at = 0;
    const int chunk = NORM_LOADS * 1024;
    rc = for_launches(items, count, chunk, [&](const AdamwLaunch &a, bool) {
        const int grid = norm_grid(a);
        if (!grid) return HGQ_OK;
        if (!parts) return fail(HGQ_ERR_ARG, "hgq_global_norm: null workspace");
        hipLaunchKernelGGL(norm_parts_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a, chunk, parts + at);
        at += grid;
        return check_launch("hgq_global_norm");
    });
    if (rc || !out) return rc;
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, parts, (int)at, out);
    return check_launch("hgq_global_norm");
}

extern "C" int hgq_adamw_update_multi(const hgq_adamw_item *items, int count, int state_bits, hgq_adamw_state *state, double beta_1,
                                      double beta_2, float epsilon, float clipnorm, double *norm_parts, int64_t n_parts, float *norm_out,
                                      uint64_t seed, const float *const *terms, int n_terms, float *sum_out, void *stream) {
    if (state_bits != 8 && state_bits != 32) return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: moments have 8 or 32 bits, not %d", state_bits);
    int rc = check_items("hgq_adamw_update_multi", items, count, state_bits);
    if (rc) return rc;
    if (!state) return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: null state");
    if (!(beta_1 >= 0 && beta_1 < 1 && beta_2 >= 0 && beta_2 < 1 && (epsilon == 0 || epsilon >= 0x1p-126f)))
        return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: 0 <= beta < 1 and an epsilon of 0 or at least 2^-126 are expected");
    if (n_parts < 0 || n_parts > 0x7fffffff || (n_parts > 0 && (!norm_parts || !(clipnorm > 0))))
        return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: a positive clipnorm and the parts of the norm go together");
    if (n_terms < 0 || n_terms > HGQ_SUM_BATCH || (n_terms > 0 && (!terms || !sum_out)))
        return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: up to %d terms and an output are expected", HGQ_SUM_BATCH);
    AdamwSum sum = {};
    sum.n = n_terms, sum.out = sum_out;
    for (int t = 0; t < n_terms; ++t)
        if (!(sum.term[t] = terms[t])) return fail(HGQ_ERR_ARG, "hgq_adamw_update_multi: null term %d", t);
    int64_t bytes = 0;
    for (int t = 0; t < count; ++t) bytes += items[t].n * ((items[t].type == HGQ_TYPE_F32 ? 12 : 6) + (state_bits == 32 ? 16 : 4));
    const bool stream_through = bytes > ADAMW_CACHE;
    // tens of thousands of workgroups take the norm, not its parts
    float *joined = nullptr;
    if (stream_through && n_parts > 0) {
        joined = norm_out ? norm_out : (float *)norm_parts;
        hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, norm_parts, (int)n_parts, joined);
        if ((rc = check_launch("hgq_adamw_update_multi"))) return rc;
        norm_out = nullptr;
    }
    return for_launches(items, count, stream_through ? ADAMW_STREAM_CHUNK : ADAMW_CHUNK, [&](const AdamwLaunch &a, bool last) {
        const uint32_t chunks = a.start[ADAMW_ITEMS], most = stream_through ? chunks : ADAMW_GRID;
        const int grid = chunks < 1 ? 1 : (int)(chunks < most ? chunks : most);  // (no element at all: the step still counts)
        auto kernel = state_bits == 8 ? stream_through ? adamw_kernel<8, true> : adamw_kernel<8, false>
                                      : stream_through ? adamw_kernel<32, true> : adamw_kernel<32, false>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, a, sum, state, beta_1, beta_2, epsilon, clipnorm, norm_parts,
                           (int)n_parts, joined, norm_out, seed, (int)last);
        sum.n = 0, norm_out = nullptr;
        return check_launch("hgq_adamw_update_multi");
    });
}
