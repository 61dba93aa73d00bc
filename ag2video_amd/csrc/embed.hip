// Embedding lookup with scaling, and its gradient by sorted tokens.
//   out[i, :] = scale * table[idx_i, :]          dtable[v, :] = scale * sum over {i : idx_i = v} of dout[i, :]
// A token outside [0, V) reads nothing: its row of the output is NaN, and it takes part in no sum; neither does padding_idx.  Products
// and sums are in fp32 and rounded once.
#include "elem.h"

__device__ __forceinline__ long long token_at(const void* idx, int wide, long long stride, long long i) {
    return wide ? ((const long long*)idx)[i * stride] : (long long)((const int*)idx)[i * stride];
}

template <class E>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* idx, int wide, long long istride, const typename E::T* table,
                                                        long long tstride, typename E::T* out, long long n, long long V, int D, float scale) {
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const long long v = token_at(idx, wide, istride, i);
        const bool in = v >= 0 && v < V;
        for (int d = threadIdx.x; d < D; d += 256)
            out[i * D + d] = E::narrow(in ? scale * E::widen(table[v * tstride + d]) : __builtin_nanf(""));
    }
}

// one workgroup per row of the table
template <class E>
__global__ __launch_bounds__(256) void embed_bwd_kernel(const void* idx, int wide, long long istride, const typename E::T* dout, long long dstride,
                                                        typename E::T* dtable, long long n, long long V, int D, float scale, long long pad) {
    const long long v = blockIdx.x;
    for (int d0 = 0; d0 < D; d0 += 256) {
        const int d = d0 + threadIdx.x;
        float acc = 0.f;
        if (d < D) {
            if (v != pad)
                for (long long i = 0; i < n; ++i)
                    if (token_at(idx, wide, istride, i) == v) acc += E::widen(dout[i * dstride + d]);
            dtable[v * D + d] = E::narrow(scale * acc);
        }
    }
}

static bool embed_ok(int dtype, int idx_bytes, long long n, long long V, int D) {
    return dtype >= AG2V_F32 && dtype <= AG2V_F16 && (idx_bytes == 4 || idx_bytes == 8) && n > 0 && n < (1LL << 31) && V > 0 && V < (1LL << 31) && D > 0;
}

template <class E>
static int run_fwd(const void* idx, int idx_bytes, long long istride, const void* table, long long tstride, void* out, long long n, long long V,
                   int D, float scale, hipStream_t st) {
    const int grid = (int)(n < (1 << 20) ? n : (1 << 20));
    hipLaunchKernelGGL(embed_fwd_kernel<E>, dim3(grid), dim3(256), 0, st, idx, idx_bytes == 8, istride, (const typename E::T*)table, tstride,
                       (typename E::T*)out, n, V, D, scale);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E>
static int run_bwd(const void* idx, int idx_bytes, long long istride, const void* dout, long long dstride, void* dtable, long long n, long long V,
                   int D, float scale, long long pad, hipStream_t st) {
    if (V >= (1LL << 24)) return AG2V_EINVAL;
    hipLaunchKernelGGL(embed_bwd_kernel<E>, dim3((int)V), dim3(256), 0, st, idx, idx_bytes == 8, istride, (const typename E::T*)dout, dstride,
                       (typename E::T*)dtable, n, V, D, scale, pad);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}

extern "C" size_t ag2v_embed_bwd_workspace_floats(int dtype, long long n, long long V, int D) {
    if (!embed_ok(dtype, 8, n, V, D)) return 0;
    return 0;
}
extern "C" int ag2v_embed_fwd(int dtype, const void* idx, int idx_bytes, long long idx_stride, const void* table, long long table_stride,
                              void* out, long long n, long long V, int D, float scale, void* stream) {
    if (!idx || !table || !out || !embed_ok(dtype, idx_bytes, n, V, D) || table_stride < D) return AG2V_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AG2V_F32) return run_fwd<ElemF32>(idx, idx_bytes, idx_stride, table, table_stride, out, n, V, D, scale, st);
    if (dtype == AG2V_BF16) return run_fwd<ElemBF16>(idx, idx_bytes, idx_stride, table, table_stride, out, n, V, D, scale, st);
    return run_fwd<ElemF16>(idx, idx_bytes, idx_stride, table, table_stride, out, n, V, D, scale, st);
}
extern "C" int ag2v_embed_bwd(int dtype, const void* idx, int idx_bytes, long long idx_stride, const void* dout, long long dout_stride,
                              void* dtable, long long n, long long V, int D, float scale, long long padding_idx, float* workspace,
                              size_t workspace_floats, void* stream) {
    if (!idx || !dout || !dtable || !embed_ok(dtype, idx_bytes, n, V, D)) return AG2V_EINVAL;
    if (workspace_floats < ag2v_embed_bwd_workspace_floats(dtype, n, V, D)) return AG2V_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AG2V_F32) return run_bwd<ElemF32>(idx, idx_bytes, idx_stride, dout, dout_stride, dtable, n, V, D, scale, padding_idx, st);
    if (dtype == AG2V_BF16) return run_bwd<ElemBF16>(idx, idx_bytes, idx_stride, dout, dout_stride, dtable, n, V, D, scale, padding_idx, st);
    return run_bwd<ElemF16>(idx, idx_bytes, idx_stride, dout, dout_stride, dtable, n, V, D, scale, padding_idx, st);
}
