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
    int act;
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

__device__ __forceinline__ float activate(float z, int act) {
    if (act == HGQ_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if (act == HGQ_ACT_SILU) return z / (1.0f + expf(-z));
    return z;
}

// dy act'(z)
__device__ __forceinline__ float through_activation(float dy, float z, int act) {
    if (act == HGQ_ACT_RELU) return z > 0.0f ? dy : z != z ? z : 0.0f;
    if (act == HGQ_ACT_SILU) {
        const float p = 1.0f / (1.0f + expf(-z));
        return dy * (p * (1.0f + z * (1.0f - p)));
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

// One workgroup per sample and group, any shape: the group is read three times, its sums are formed in fp64.
template <typename T>
__global__ __launch_bounds__(256) void group_norm_fwd_any(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                                          T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out, GroupShape s) {
    __shared__ double lds[4];
    const int64_t b = blockIdx.x / s.G;
    const int g = (int)(blockIdx.x % s.G);
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
    if (threadIdx.x == 0) mean_out[blockIdx.x] = mean, rstd_out[blockIdx.x] = rstd;
    for (int64_t e = threadIdx.x; e < n; e += 256) {
        const int c = g * s.D + (int)(e % s.D);
        const int64_t at = base + e / s.D * s.C + e % s.D;
        const float z = (to_f32(x[at]) - mean) * rstd * (gamma ? gamma[c] : 1.0f) + (beta ? beta[c] : 0.0f);
        y[at] = (T)activate(z, s.act);
    }
}

// One workgroup per sample and group, any shape.  part [B][2 C]: each sample's terms of dgamma, then of dbeta.
template <typename T>
__global__ __launch_bounds__(256) void group_norm_bwd_any(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                          const float *__restrict__ beta, const float *__restrict__ mean_in,
                                                          const float *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ part, GroupShape s) {
    __shared__ double lds[4];
    __shared__ double col[2][256];
    const int64_t b = blockIdx.x / s.G;
    const int g = (int)(blockIdx.x % s.G);
    const int64_t base = b * s.S * s.C + (int64_t)g * s.D, n = s.S * s.D;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    int tx = 1;  // threads side by side over channels, the others over positions
    while (tx < s.D && tx < 256) tx *= 2;
    const int ty = 256 / tx, cx = threadIdx.x % tx, py = threadIdx.x / tx;
    double s1 = 0, s2 = 0;  // of d and d xhat, over the group
    for (int c0 = 0; c0 < s.D; c0 += tx) {
        const int d = c0 + cx, c = g * s.D + d;
        double a = 0, h = 0;
        const float ga = d < s.D && gamma ? gamma[c] : 1.0f, be = d < s.D && beta ? beta[c] : 0.0f;
        if (d < s.D)
            for (int64_t p = py; p < s.S; p += ty) {
                const int64_t at = base + p * s.C + d;
                const float xh = (to_f32(x[at]) - mean) * rstd;
                const float dz = through_activation(to_f32(dy[at]), xh * ga + be, s.act);
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
    if (!dx) return;
    for (int64_t e = threadIdx.x; e < n; e += 256) {
        const int c = g * s.D + (int)(e % s.D);
        const int64_t at = base + e / s.D * s.C + e % s.D;
        const float ga = gamma ? gamma[c] : 1.0f, xh = (to_f32(x[at]) - mean) * rstd;
        const float dz = through_activation(to_f32(dy[at]), xh * ga + (beta ? beta[c] : 0.0f), s.act);
        dx[at] = (T)((dz * ga - m1 - xh * m2) * rstd);
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

template <typename T>
int fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, const GroupShape &s, hipStream_t st) {
    hipLaunchKernelGGL(group_norm_fwd_any<T>, dim3((unsigned)(s.B * s.G)), dim3(256), 0, st, (const T *)x, gamma, beta, (T *)y, mean, rstd, s);
    return check_launch("hgq_group_norm_fwd");
}

template <typename T>
int bwd(const void *dy, const void *x, const float *gamma, const float *beta, const float *mean, const float *rstd, void *dx, float *dgamma,
        float *dbeta, float *ws, const GroupShape &s, hipStream_t st) {
    const bool sums = dgamma || dbeta;
    hipLaunchKernelGGL(group_norm_bwd_any<T>, dim3((unsigned)(s.B * s.G)), dim3(256), 0, st, (const T *)dy, (const T *)x, gamma, beta, mean, rstd, (T *)dx,
                       sums ? ws : nullptr, s);
    const int rc = check_launch("hgq_group_norm_bwd");
    if (rc || !sums) return rc;
    return reduce_parts(ws, (int)s.B, 2 * (int64_t)s.C, dgamma, s.C, dbeta, s.C, nullptr, 0, st);
}

}  // namespace

extern "C" int64_t hgq_group_norm_fwd_workspace(int64_t B, int64_t S, int C, int G, int type) {
    return check_shape("hgq_group_norm_fwd_workspace", B, S, C, G, HGQ_ACT_NONE, type) ? -1 : 0;
}

extern "C" int64_t hgq_group_norm_bwd_workspace(int64_t B, int64_t S, int C, int G, int type) {
    return check_shape("hgq_group_norm_bwd_workspace", B, S, C, G, HGQ_ACT_NONE, type) ? -1 : B * 2 * C;
}

extern "C" int hgq_group_norm_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, float *workspace,
                                  int64_t B, int64_t S, int C, int G, float eps, int act, int type, void *stream) {
    int rc = check_shape("hgq_group_norm_fwd", B, S, C, G, act, type);
    if (rc) return rc;
    if (!(eps >= 0)) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: epsilon must not be negative");
    if (B == 0 || S == 0) return HGQ_OK;
    if (!x || !y || !mean || !rstd) return fail(HGQ_ERR_ARG, "hgq_group_norm_fwd: null pointer");
    const GroupShape s = {B, S, C, G, C / G, eps, act};
    return (type == HGQ_TYPE_F32 ? fwd<float> : type == HGQ_TYPE_BF16 ? fwd<__bf16> : fwd<_Float16>)(x, gamma, beta, y, mean, rstd, s, (hipStream_t)stream);
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
    const GroupShape s = {B, S, C, G, C / G, 0.0f, act};
    return (type == HGQ_TYPE_F32 ? bwd<float> : type == HGQ_TYPE_BF16 ? bwd<__bf16> : bwd<_Float16>)(dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, workspace, s,
                                                                                                    (hipStream_t)stream);
}
