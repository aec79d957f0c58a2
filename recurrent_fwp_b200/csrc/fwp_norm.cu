// Norms between two blocks, forward (see fwp_norm.cuh).
#include "fwp_norm.cuh"

namespace fwp {

template <int TPR, int EPT, int V>
__device__ __forceinline__ void row_statistics(const float (&v)[EPT], const NormParams& p, int tid, float* buf, float& mean, float& rstd) {
    mean = 0.f;
    constexpr int W = TPR / 32;
    if (!p.rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < EPT; i++) s[0] += v[i];         // elements beyond the row are zero
        row_sum<TPR, 1>(s, buf);
        mean = s[0] / p.D;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < EPT; i++) {
        const float c = row_has<TPR, V>(i, p.D, tid) ? v[i] - mean : 0.f;
        q[0] = fmaf(c, c, q[0]);
    }
    row_sum<TPR, 1>(q, buf + W);
    rstd = rsqrtf(q[0] / p.D + p.eps);
}

template <typename T, typename TR, int TPR, int EPT, int V>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_fwd_kernel(NormParams p) {
    __shared__ float buf[TPR > 32 ? TPR / 32 * 4 : 1];
    griddep_wait();
    griddep_launch_dependents();
    constexpr int RPC = TPR == 32 ? 4 : 1;
    const int tid = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * RPC + threadIdx.x / TPR;
    if (row >= p.rows) return;
    const long long n = row / p.L, l = row - n * p.L;
    auto at = [&](const Stream& s) { return n * s.sN + l * s.sL; };
    float x[EPT], r[EPT], g[EPT];
    row_load<TPR, EPT, V>(static_cast<const T*>(p.x.p) + at(p.x), p.D, tid, x);
    if (p.res.p) row_load<TPR, EPT, V>(static_cast<const TR*>(p.res.p) + at(p.res), p.D, tid, r);
    if (p.gate.p) row_load<TPR, EPT, V>(static_cast<const T*>(p.gate.p) + at(p.gate), p.D, tid, g);
    float stats[4] = {0.f, 1.f, 0.f, 1.f};
    if (p.pw) {
        row_statistics<TPR, EPT, V>(x, p, tid, buf, stats[0], stats[1]);
        float w[EPT], b[EPT];
        row_load<TPR, EPT, V>(p.pw, p.D, tid, w);
        if (p.pb) row_load<TPR, EPT, V>(p.pb, p.D, tid, b);
#pragma unroll
        for (int i = 0; i < EPT; i++) x[i] = fmaf((x[i] - stats[0]) * stats[1], w[i], p.pb ? b[i] : 0.f);
    }
    if (p.gate.p)
#pragma unroll
        for (int i = 0; i < EPT; i++) x[i] *= gate_of(p.act, g[i]);
    if (p.sv) {
        row_load<TPR, EPT, V>(p.sv, p.D, tid, g);
#pragma unroll
        for (int i = 0; i < EPT; i++) x[i] *= g[i];
    } else {
#pragma unroll
        for (int i = 0; i < EPT; i++) x[i] *= p.sval;
    }
#pragma unroll
    for (int i = 0; i < EPT; i++) {
        if (p.res.p) x[i] += r[i];
        if (!row_has<TPR, V>(i, p.D, tid)) x[i] = 0.f;
    }
    row_store<TPR, EPT, V>(static_cast<TR*>(p.r.p) + at(p.r), p.D, tid, x);
    row_statistics<TPR, EPT, V>(x, p, tid, buf + (TPR > 32 ? TPR / 16 : 0), stats[2], stats[3]);
    row_load<TPR, EPT, V>(p.w, p.D, tid, g);
    if (p.b) row_load<TPR, EPT, V>(p.b, p.D, tid, r);
#pragma unroll
    for (int i = 0; i < EPT; i++) x[i] = fmaf((x[i] - stats[2]) * stats[3], g[i], p.b ? r[i] : 0.f);
    row_store<TPR, EPT, V>(static_cast<T*>(p.y.p) + at(p.y), p.D, tid, x);
    if (p.stats && tid == 0) *reinterpret_cast<float4*>(p.stats + 4 * row) = make_float4(stats[0], stats[1], stats[2], stats[3]);
}

template <typename T, typename TR, int TPR, int EPT>
static int norm_launch(const NormParams& p, bool vec, cudaStream_t st) {
    constexpr int RPC = TPR == 32 ? 4 : 1, threads = TPR == 32 ? 128 : TPR;
    const long long ctas = ceil_div(p.rows, RPC);
    if (ctas > 0x7fffffffLL) return FWP_ERR_SHAPE;
    if (vec) return launch_dependent(norm_fwd_kernel<T, TR, TPR, EPT, 4>, p, dim3((unsigned)ctas), threads, 0, st, "norm_fwd_kernel");
    return launch_dependent(norm_fwd_kernel<T, TR, TPR, EPT, 1>, p, dim3((unsigned)ctas), threads, 0, st, "norm_fwd_kernel");
}
template <typename T, typename TR>
static int norm_dispatch(const NormParams& p, bool vec, cudaStream_t st) {
    if (p.D <= 128) return norm_launch<T, TR, 32, 4>(p, vec, st);
    if (p.D <= 256) return norm_launch<T, TR, 32, 8>(p, vec, st);
    if (p.D <= 512) return norm_launch<T, TR, 32, 16>(p, vec, st);
    if (p.D <= 1024) return norm_launch<T, TR, 128, 8>(p, vec, st);
    if (p.D <= 2048) return norm_launch<T, TR, 128, 16>(p, vec, st);
    if (p.D <= 4096) return norm_launch<T, TR, 256, 16>(p, vec, st);
    return norm_launch<T, TR, 512, 16>(p, vec, st);
}

}  // namespace fwp

using namespace fwp;

FWP_API int fwp_block_norm_forward(int N, int L, int D, const fwp_tensor* x, const fwp_tensor* residual, const fwp_tensor* gate,
                                   const float* scale_vector, float scale_value, const float* post_weight, const float* post_bias,
                                   const float* weight, const float* bias, const fwp_tensor* y, const fwp_tensor* r, float* stats,
                                   float eps, int rms, int gate_act, int io_dtype, int residual_dtype, void* stream, int device) {
    int rc;
    if ((rc = norm_check(N, L, D, x, residual, gate, scale_vector, post_weight, post_bias, weight, bias, gate_act, io_dtype, residual_dtype)))
        return rc;
    const int esz = io_dtype == FWP_F32 ? 4 : 2, rsz = residual_dtype == FWP_F32 ? 4 : 2;
    if (!N || !L || !D) return FWP_OK;
    if ((rc = check_tensor(y, esz, true)) || (rc = check_tensor(r, rsz, true))) return rc;
    if (!aligned16(stats)) return FWP_ERR_ALIGN;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    NormParams p = norm_params(N, L, D, x, residual, gate, scale_vector, scale_value, post_weight, post_bias, weight, bias, rms, gate_act);
    p.y = stream_of(y);
    p.r = stream_of(r);
    p.stats = stats;
    p.eps = eps;
    const bool vec = norm_vectors(p) && rows_aligned(p.x, esz, 4 * esz) && rows_aligned(p.res, rsz, 4 * rsz) && rows_aligned(p.gate, esz, 4 * esz) &&
                     rows_aligned(p.y, esz, 4 * esz) && rows_aligned(p.r, rsz, 4 * rsz);
    cudaStream_t st = (cudaStream_t)stream;
    if (io_dtype == FWP_F32) return norm_dispatch<float, float>(p, vec, st);
    if (residual_dtype == FWP_F32) return norm_dispatch<__nv_bfloat16, float>(p, vec, st);
    return norm_dispatch<__nv_bfloat16, __nv_bfloat16>(p, vec, st);
}
