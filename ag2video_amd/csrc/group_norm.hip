// Group norm with an activation on channels-last maps, forward and backward.
//   x[N, S, C], G groups of Cg = C / G channels, M = S * Cg values per (sample, group):
//     h = (x - mean) * rstd      mean, biased variance over the group's S positions and Cg channels, rstd = 1 / sqrt(var + eps)
//     z = w h + b                y = act(z):  0 z,  1 z * sigmoid(z),  2 z > 0 ? z : slope * z
//   backward, dz = dy act'(z), A[n,c] = sum_s dz, B[n,c] = sum_s dz h:
//     db = sum_n A, dw = sum_n B, s1 = sum_{c in g} w A, s2 = sum_{c in g} w B, dx = rstd (w dz - (s1 + h s2) / M)
// Every sum is in fp32; z and h are computed again in the backward pass from x and the two statistics of a group.
#include "elem.h"

#define ACT_NONE 0
#define ACT_SILU 1
#define ACT_LRELU 2

struct GnArgs {
    const void *x, *dy, *w, *b;
    void *y, *dw, *db;
    float *mean, *rstd;
    long long xs, xr, ds, dr;   // strides of x and dy in elements: between samples, between positions (channels are adjacent)
    int N, S, C, G, Cg, ptype;
    float eps, slope;
};

template <int ACT>
__device__ __forceinline__ float act_fwd(float z, float slope) {
    if (ACT == ACT_SILU) return z * __frcp_rn(1.f + __expf(-z));
    if (ACT == ACT_LRELU) return z > 0.f ? z : z * slope;
    return z;
}
// dy * act'(z)
template <int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z, float slope) {
    if (ACT == ACT_SILU) {
        const float s = __frcp_rn(1.f + __expf(-z));
        return dy * (s * (1.f + z * (1.f - s)));
    }
    if (ACT == ACT_LRELU) return z > 0.f ? dy : dy * slope;
    return dy;
}

// one workgroup per (sample, group), three passes over its values
template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_fwd_kernel(GnArgs a) {
    __shared__ float sh[4];
    const int n = blockIdx.x / a.G, g = blockIdx.x - n * a.G;
    const long long M = (long long)a.S * a.Cg;
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + g * a.Cg;
    typename E::T* y = (typename E::T*)a.y + (long long)n * a.S * a.C + g * a.Cg;
    float s = 0.f;
    for (long long e = threadIdx.x; e < M; e += 256) s += E::widen(x[e / a.Cg * a.xr + e % a.Cg]);
    const float mean = block_sum_256(s, sh) / (float)M;
    float m2 = 0.f;
    for (long long e = threadIdx.x; e < M; e += 256) {
        const float d = E::widen(x[e / a.Cg * a.xr + e % a.Cg]) - mean;
        m2 += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum_256(m2, sh) / (float)M + a.eps);
    if (threadIdx.x == 0) { a.mean[blockIdx.x] = mean; a.rstd[blockIdx.x] = rstd; }
    for (long long e = threadIdx.x; e < M; e += 256) {
        const long long r = e / a.Cg;
        const int c = (int)(e - r * a.Cg);
        const float w = a.w ? load_any(a.w, a.ptype, g * a.Cg + c) : 1.f, b = a.b ? load_any(a.b, a.ptype, g * a.Cg + c) : 0.f;
        const float h = (E::widen(x[r * a.xr + c]) - mean) * rstd;
        y[r * a.C + c] = E::narrow(act_fwd<ACT>(h * w + b, a.slope));
    }
}

template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_dx_kernel(GnArgs a) {
    __shared__ float sh[4];
    const int n = blockIdx.x / a.G, g = blockIdx.x - n * a.G;
    const long long M = (long long)a.S * a.Cg;
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + g * a.Cg;
    const typename E::T* dy = (const typename E::T*)a.dy + n * a.ds + g * a.Cg;
    typename E::T* dx = (typename E::T*)a.y + (long long)n * a.S * a.C + g * a.Cg;
    const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
    float s1 = 0.f, s2 = 0.f;
    for (long long e = threadIdx.x; e < M; e += 256) {
        const long long r = e / a.Cg;
        const int c = (int)(e - r * a.Cg);
        const float w = a.w ? load_any(a.w, a.ptype, g * a.Cg + c) : 1.f, b = a.b ? load_any(a.b, a.ptype, g * a.Cg + c) : 0.f;
        const float h = (E::widen(x[r * a.xr + c]) - mean) * rstd;
        const float t = w * act_bwd<ACT>(E::widen(dy[r * a.dr + c]), h * w + b, a.slope);
        s1 += t;
        s2 += t * h;
    }
    s1 = block_sum_256(s1, sh) / (float)M;
    s2 = block_sum_256(s2, sh) / (float)M;
    for (long long e = threadIdx.x; e < M; e += 256) {
        const long long r = e / a.Cg;
        const int c = (int)(e - r * a.Cg);
        const float w = a.w ? load_any(a.w, a.ptype, g * a.Cg + c) : 1.f, b = a.b ? load_any(a.b, a.ptype, g * a.Cg + c) : 0.f;
        const float h = (E::widen(x[r * a.xr + c]) - mean) * rstd;
        const float t = w * act_bwd<ACT>(E::widen(dy[r * a.dr + c]), h * w + b, a.slope);
        dx[r * a.C + c] = E::narrow(rstd * (t - s1 - h * s2));
    }
}

// one workgroup per channel
template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_params_kernel(GnArgs a) {
    __shared__ float sh[4];
    const int c = blockIdx.x, g = c / a.Cg;
    const typename E::T* x = (const typename E::T*)a.x + c;
    const typename E::T* dy = (const typename E::T*)a.dy + c;
    const float w = a.w ? load_any(a.w, a.ptype, c) : 1.f, b = a.b ? load_any(a.b, a.ptype, c) : 0.f;
    float A = 0.f, B = 0.f;
    for (long long e = threadIdx.x; e < (long long)a.N * a.S; e += 256) {
        const long long n = e / a.S, r = e - n * a.S;
        const float h = (E::widen(x[n * a.xs + r * a.xr]) - a.mean[n * a.G + g]) * a.rstd[n * a.G + g];
        const float dz = act_bwd<ACT>(E::widen(dy[n * a.ds + r * a.dr]), h * w + b, a.slope);
        A += dz;
        B += dz * h;
    }
    A = block_sum_256(A, sh);
    B = block_sum_256(B, sh);
    if (threadIdx.x == 0) {
        if (a.dw) store_any(a.dw, a.ptype, c, B);
        if (a.db) store_any(a.db, a.ptype, c, A);
    }
}

template <class E, int ACT>
static int run_fwd(const GnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((gn_fwd_kernel<E, ACT>), dim3(a.N * a.G), dim3(256), 0, st, a);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT>
static int run_bwd(const GnArgs& a, hipStream_t st) {
    if (a.y) hipLaunchKernelGGL((gn_bwd_dx_kernel<E, ACT>), dim3(a.N * a.G), dim3(256), 0, st, a);
    AG2V_CHECK_LAUNCH();
    if (a.dw || a.db) hipLaunchKernelGGL((gn_bwd_params_kernel<E, ACT>), dim3(a.C), dim3(256), 0, st, a);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E>
static int run_elem(const GnArgs& a, int act, bool backward, hipStream_t st) {
    if (act == ACT_SILU) return backward ? run_bwd<E, ACT_SILU>(a, st) : run_fwd<E, ACT_SILU>(a, st);
    if (act == ACT_LRELU) return backward ? run_bwd<E, ACT_LRELU>(a, st) : run_fwd<E, ACT_LRELU>(a, st);
    return backward ? run_bwd<E, ACT_NONE>(a, st) : run_fwd<E, ACT_NONE>(a, st);
}
static int run_any(const GnArgs& a, int dtype, int act, bool backward, hipStream_t st) {
    if (dtype == AG2V_F32) return run_elem<ElemF32>(a, act, backward, st);
    return dtype == AG2V_BF16 ? run_elem<ElemBF16>(a, act, backward, st) : run_elem<ElemF16>(a, act, backward, st);
}

static bool sizes_ok(int dtype, int ptype, int N, int S, int C, int groups, int act) {
    if (dtype < AG2V_F32 || dtype > AG2V_F16 || ptype < AG2V_F32 || ptype > AG2V_F16 || act < ACT_NONE || act > ACT_LRELU) return false;
    if (N <= 0 || S <= 0 || C <= 0 || groups <= 0 || C % groups) return false;
    return (long long)N * groups < (1LL << 31);
}

extern "C" size_t ag2v_group_norm_workspace_floats(int dtype, int N, int S, int C, int groups, int backward) {
    if (!sizes_ok(dtype, AG2V_F32, N, S, C, groups, ACT_NONE)) return 0;
    return 0;
}
extern "C" int ag2v_group_norm_fwd(int dtype, const void* x, long long x_sample, long long x_row, const void* weight, const void* bias,
                                   int param_dtype, void* y, float* mean, float* rstd, int N, int S, int C, int groups, float eps, int act,
                                   float slope, float* workspace, size_t workspace_floats, void* stream) {
    if (!x || !y || !mean || !rstd || !sizes_ok(dtype, param_dtype, N, S, C, groups, act) || !(eps >= 0.f)) return AG2V_EINVAL;
    if (workspace_floats < ag2v_group_norm_workspace_floats(dtype, N, S, C, groups, 0)) return AG2V_EINVAL;
    GnArgs a = {};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd; a.xs = x_sample; a.xr = x_row;
    a.N = N; a.S = S; a.C = C; a.G = groups; a.Cg = C / groups; a.ptype = param_dtype; a.eps = eps; a.slope = slope;
    return run_any(a, dtype, act, false, (hipStream_t)stream);
}
extern "C" int ag2v_group_norm_bwd(int dtype, const void* dy, long long dy_sample, long long dy_row, const void* x, long long x_sample,
                                   long long x_row, const void* weight, const void* bias, int param_dtype, const float* mean,
                                   const float* rstd, void* dx, void* dweight, void* dbias, int N, int S, int C, int groups, int act,
                                   float slope, float* workspace, size_t workspace_floats, void* stream) {
    if (!x || !dy || !mean || !rstd || !sizes_ok(dtype, param_dtype, N, S, C, groups, act)) return AG2V_EINVAL;
    if (workspace_floats < ag2v_group_norm_workspace_floats(dtype, N, S, C, groups, 1)) return AG2V_EINVAL;
    GnArgs a = {};
    a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.y = dx; a.dw = dweight; a.db = dbias; a.mean = (float*)mean; a.rstd = (float*)rstd;
    a.xs = x_sample; a.xr = x_row; a.ds = dy_sample; a.dr = dy_row;
    a.N = N; a.S = S; a.C = C; a.G = groups; a.Cg = C / groups; a.ptype = param_dtype; a.slope = slope;
    return run_any(a, dtype, act, true, (hipStream_t)stream);
}
