// Norms between two blocks, backward (see fwp_norm.cuh).  With n = (r - mean) / sd, gn = gy w:
//
//   g = (gn - n mean(gn n) - mean(gn)) / sd + gr  (without the last mean for rms),  gresidual = g,  gu = s g
//   ggate = gu t act'(gate),  gt = gu act(gate),  and the same rule once more for the norm behind the block
//
// The gradients of the weights are sums over rows: a CTA walks many rows and keeps its sums in registers, the CTAs' sums are added in
// a fixed order.
#include "fwp_norm.cuh"

namespace fwp {

constexpr int norm_bwd_warps(int TPR) { return TPR == 32 ? 8 : TPR / 32; }

// FULL: with a norm behind the block, a gate or a scale vector; without, only r = residual + number x
template <typename T, typename TR, int TPR, int EPT, int V, bool FULL>
__global__ void __launch_bounds__(norm_bwd_warps(TPR) * 32) norm_bwd_kernel(NormParams p) {
    constexpr int SLOTS = TPR == 32 ? 8 : 1, NV = FULL ? 5 : 2, W = TPR / 32;
    __shared__ float buf[TPR > 32 ? 8 * W : 1];
    __shared__ float red[SLOTS > 1 ? SLOTS : 1][SLOTS > 1 ? TPR * EPT : 1];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    float acc[NV][EPT];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < EPT; i++) acc[k][i] = 0.f;
    const float inv = 1.f / p.D;
    int par = 0;
    for (long long row = (long long)blockIdx.x * SLOTS + slot; row < p.rows; row += (long long)gridDim.x * SLOTS, par ^= 1) {
        const long long n = row / p.L, l = row - n * p.L;
        auto at = [&](const Stream& s) { return n * s.sN + l * s.sL; };
        const float4 stats = *reinterpret_cast<const float4*>(p.stats + 4 * row);
        float x[EPT], r[EPT], g[EPT], gate[FULL ? EPT : 1], sc[FULL ? EPT : 1];
        row_load<TPR, EPT, V>(static_cast<const T*>(p.x.p) + at(p.x), p.D, tid, x);
#pragma unroll
        for (int i = 0; i < EPT; i++) r[i] = g[i] = 0.f;
        if (p.res.p) row_load<TPR, EPT, V>(static_cast<const TR*>(p.res.p) + at(p.res), p.D, tid, r);
        if (p.gy.p) row_load<TPR, EPT, V>(static_cast<const T*>(p.gy.p) + at(p.gy), p.D, tid, g);
        float t[FULL ? EPT : 1];        // what the gate multiplies
        if constexpr (FULL) {
            if (p.gate.p) row_load<TPR, EPT, V>(static_cast<const T*>(p.gate.p) + at(p.gate), p.D, tid, gate);
            if (p.sv) row_load<TPR, EPT, V>(p.sv, p.D, tid, sc);
            else
#pragma unroll
                for (int i = 0; i < EPT; i++) sc[i] = p.sval;
            if (p.pw) {
                row_load<TPR, EPT, V>(p.pw, p.D, tid, t);
                float b[EPT];
                if (p.pb) row_load<TPR, EPT, V>(p.pb, p.D, tid, b);
#pragma unroll
                for (int i = 0; i < EPT; i++) {
                    x[i] = row_has<TPR, V>(i, p.D, tid) ? (x[i] - stats.x) * stats.y : 0.f;
                    t[i] = fmaf(x[i], t[i], p.pb ? b[i] : 0.f);
                }
            } else {
#pragma unroll
                for (int i = 0; i < EPT; i++) t[i] = x[i];
            }
        }
        float s[2] = {0.f, 0.f}, w[EPT];
        row_load<TPR, EPT, V>(p.w, p.D, tid, w);
#pragma unroll
        for (int i = 0; i < EPT; i++) {
            float u;
            if constexpr (FULL) u = sc[i] * (p.gate.p ? t[i] * gate_of(p.act, gate[i]) : t[i]);
            else u = p.sval * x[i];
            r[i] = row_has<TPR, V>(i, p.D, tid) ? (r[i] + u - stats.z) * stats.w : 0.f;
            acc[0][i] = fmaf(g[i], r[i], acc[0][i]);
            acc[1][i] += g[i];
            g[i] *= w[i];
            s[0] = fmaf(g[i], r[i], s[0]);
            s[1] += g[i];
        }
        row_sum<TPR, 2>(s, buf + par * 4 * W);
        const float m1 = s[0] * inv, m0 = p.rms ? 0.f : s[1] * inv;
        if (p.gr.p) row_load<TPR, EPT, V>(static_cast<const TR*>(p.gr.p) + at(p.gr), p.D, tid, w);
#pragma unroll
        for (int i = 0; i < EPT; i++) g[i] = fmaf(stats.w, g[i] - r[i] * m1 - m0, p.gr.p ? w[i] : 0.f);
        if (p.gres.p) row_store<TPR, EPT, V>(static_cast<TR*>(p.gres.p) + at(p.gres), p.D, tid, g);
        if constexpr (FULL) {
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                const bool in = row_has<TPR, V>(i, p.D, tid);
                const float a = p.gate.p ? gate_of(p.act, gate[i]) : 1.f;
                if (in) acc[4][i] = fmaf(g[i], t[i] * a, acc[4][i]);
                g[i] *= sc[i];
                if (p.gate.p) gate[i] = g[i] * t[i] * gate_grad_of(p.act, gate[i]);
                g[i] = in ? g[i] * a : 0.f;
            }
            if (p.ggate.p) row_store<TPR, EPT, V>(static_cast<T*>(p.ggate.p) + at(p.ggate), p.D, tid, gate);
            if (p.pw) {
                row_load<TPR, EPT, V>(p.pw, p.D, tid, w);
                s[0] = s[1] = 0.f;
#pragma unroll
                for (int i = 0; i < EPT; i++) {
                    acc[2][i] = fmaf(g[i], x[i], acc[2][i]);
                    acc[3][i] += g[i];
                    g[i] *= w[i];
                    s[0] = fmaf(g[i], x[i], s[0]);
                    s[1] += g[i];
                }
                row_sum<TPR, 2>(s, buf + par * 4 * W + 2 * W);
                const float q1 = s[0] * inv, q0 = p.rms ? 0.f : s[1] * inv;
#pragma unroll
                for (int i = 0; i < EPT; i++) g[i] = stats.y * (g[i] - x[i] * q1 - q0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPT; i++) g[i] *= p.sval;
        }
        if (p.gx.p) row_store<TPR, EPT, V>(static_cast<T*>(p.gx.p) + at(p.gx), p.D, tid, g);
    }
    float* part = p.part + (long long)blockIdx.x * p.D * NV;
    if constexpr (SLOTS == 1) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                const int c = ((i / V) * TPR + tid) * V + i % V;
                if (c < p.D) part[(long long)k * p.D + c] = acc[k][i];
            }
    } else {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < EPT; i++) red[slot][((i / V) * TPR + tid) * V + i % V] = acc[k][i];
            __syncthreads();
            for (int c = threadIdx.x; c < p.D; c += SLOTS * TPR) {
                float a = 0.f;
#pragma unroll
                for (int q = 0; q < SLOTS; q++) a += red[q][c];
                part[(long long)k * p.D + c] = a;
            }
        }
    }
}

// CTAs: enough warps to keep the memory busy, and no more partial sums than that
static int norm_bwd_ctas(long long rows, int D) {
    const long long sms = sm_count() > 0 ? sm_count() : 148;
    const long long per_sm = D <= 1024 ? 4 : D <= 2048 ? 3 : D <= 4096 ? 2 : 1;
    const long long most = D <= 256 ? ceil_div(rows, 8) : rows;
    return (int)(most < sms * per_sm ? most : sms * per_sm);
}

template <typename T, typename TR, int TPR, int EPT, bool FULL>
static int norm_bwd_launch(const NormParams& p, bool vec, int ctas, cudaStream_t st) {
    constexpr int threads = norm_bwd_warps(TPR) * 32;
    if (vec) return launch_dependent(norm_bwd_kernel<T, TR, TPR, EPT, 4, FULL>, p, dim3(ctas), threads, 0, st, "norm_bwd_kernel");
    return launch_dependent(norm_bwd_kernel<T, TR, TPR, EPT, 1, FULL>, p, dim3(ctas), threads, 0, st, "norm_bwd_kernel");
}
template <typename T, typename TR, bool FULL>
static int norm_bwd_dispatch(const NormParams& p, bool vec, int ctas, cudaStream_t st) {
    if (p.D <= 256) return norm_bwd_launch<T, TR, 32, 8, FULL>(p, vec, ctas, st);
    if (p.D <= 512) return norm_bwd_launch<T, TR, 64, 8, FULL>(p, vec, ctas, st);
    if (p.D <= 1024) return norm_bwd_launch<T, TR, 128, 8, FULL>(p, vec, ctas, st);
    if (p.D <= 2048) return norm_bwd_launch<T, TR, 256, 8, FULL>(p, vec, ctas, st);
    if (p.D <= 4096) return norm_bwd_launch<T, TR, 512, 8, FULL>(p, vec, ctas, st);
    return norm_bwd_launch<T, TR, 1024, 8, FULL>(p, vec, ctas, st);
}

}  // namespace fwp

using namespace fwp;

FWP_API int64_t fwp_block_norm_backward_scratch_floats(int N, int L, int D) {
    if (N <= 0 || L <= 0 || D <= 0 || D > kNormMaxD) return 0;
    return (int64_t)norm_bwd_ctas((long long)N * L, D) * D * 5;
}

FWP_API int fwp_block_norm_backward(int N, int L, int D, const fwp_tensor* x, const fwp_tensor* residual, const fwp_tensor* gate,
                                    const float* scale_vector, float scale_value, const float* post_weight, const float* post_bias,
                                    const float* weight, const float* bias, const float* stats, const fwp_tensor* grad_y,
                                    const fwp_tensor* grad_r, const fwp_tensor* grad_x, const fwp_tensor* grad_residual,
                                    const fwp_tensor* grad_gate, float* grad_scale, float* grad_post_weight, float* grad_post_bias,
                                    float* grad_weight, float* grad_bias, float* scratch, int64_t scratch_floats, int rms, int gate_act,
                                    int io_dtype, int residual_dtype, void* stream, int device) {
    int rc;
    if ((rc = norm_check(N, L, D, x, residual, gate, scale_vector, post_weight, post_bias, weight, bias, gate_act, io_dtype, residual_dtype)))
        return rc;
    const int esz = io_dtype == FWP_F32 ? 4 : 2, rsz = residual_dtype == FWP_F32 ? 4 : 2;
    if (N && L && D && ((rc = check_tensor(grad_y, esz, false)) || (rc = check_tensor(grad_r, rsz, false)) || (rc = check_tensor(grad_x, esz, true)) ||
        (rc = check_tensor(grad_residual, rsz, false)) || (rc = check_tensor(grad_gate, esz, given(gate)))))
        return rc;
    if (D && !grad_weight) return FWP_ERR_NULL;
    for (const float* q : {(const float*)grad_scale, (const float*)grad_post_weight, (const float*)grad_post_bias, (const float*)grad_weight, (const float*)grad_bias})
        if (!aligned4(q)) return FWP_ERR_ALIGN;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    cudaStream_t st = (cudaStream_t)stream;
    if (!N || !L || !D) {               // no rows: sums of nothing
        cudaError_t e = cudaSuccess;
        for (float* q : {grad_scale, grad_post_weight, grad_post_bias, grad_weight, grad_bias})
            if (q && D && e == cudaSuccess) e = cudaMemsetAsync(q, 0, sizeof(float) * D, st);
        return e == cudaSuccess ? FWP_OK : set_cuda_error(e);
    }
    if (!stats) return FWP_ERR_NULL;
    if (!aligned16(stats)) return FWP_ERR_ALIGN;
    if (!scratch || !aligned16(scratch) || scratch_floats < fwp_block_norm_backward_scratch_floats(N, L, D)) return FWP_ERR_SCRATCH;
    NormParams p = norm_params(N, L, D, x, residual, gate, scale_vector, scale_value, post_weight, post_bias, weight, bias, rms, gate_act);
    p.gy = stream_of(grad_y); p.gr = stream_of(grad_r); p.gx = stream_of(grad_x); p.gres = stream_of(grad_residual);
    p.ggate = stream_of(grad_gate);
    p.stats = const_cast<float*>(stats);
    p.part = scratch;
    bool vec = norm_vectors(p);
    for (const Stream* s : {&p.x, &p.gate, &p.gy, &p.gx, &p.ggate}) vec = vec && rows_aligned(*s, esz, 4 * esz);
    for (const Stream* s : {&p.res, &p.gr, &p.gres}) vec = vec && rows_aligned(*s, rsz, 4 * rsz);
    const bool full = p.pw || p.gate.p || p.sv;
    const int ctas = norm_bwd_ctas(p.rows, D);
    auto run = [&](auto t, auto r) {
        using T = decltype(t);
        using TR = decltype(r);
        return full ? norm_bwd_dispatch<T, TR, true>(p, vec, ctas, st) : norm_bwd_dispatch<T, TR, false>(p, vec, ctas, st);
    };
    if (io_dtype == FWP_F32) rc = run(float(), float());
    else if (residual_dtype == FWP_F32) rc = run(__nv_bfloat16(), float());
    else rc = run(__nv_bfloat16(), __nv_bfloat16());
    if (rc) return rc;
    ColumnSums s = {scratch, ctas, (long long)D * (full ? 5 : 2), {grad_weight, grad_bias, grad_post_weight, grad_post_bias, grad_scale}, {}};
    for (int k = 0; k < kSumSegments; k++) s.end[k] = (long long)D * (k + 1);
    return launch_column_sums(s, st);
}
