// Norms between two blocks, forward (see fwp_norm.cuh).
#include "fwp_norm.cuh"

namespace fwp {

// (v - mean) / sd with the mean zero for rms; the variance is taken around the mean
template <int TPR, int EPT, int V>
__device__ __forceinline__ void row_normalise(f2 (&v)[EPT / 2], const NormParams& p, int tid, float* buf, float& mean, float& rstd) {
    constexpr int W = TPR / 32;
    mean = 0.f;
    if (!p.rms) {
        f2 a = v[0];
#pragma unroll
        for (int i = 1; i < EPT / 2; i++) a = fadd2(a, v[i]);
        float s[1] = {f2_hsum(a)};
        row_sum<TPR, 1>(s, buf);
        mean = s[0] / p.D;
        const f2 m = f2_all(-mean);
#pragma unroll
        for (int i = 0; i < EPT / 2; i++) v[i] = fadd2(v[i], m);
        row_cut<TPR, EPT, V>(p.D, tid, v);
    }
    f2 q = fmul2(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < EPT / 2; i++) q = ffma2(v[i], v[i], q);
    float s[1] = {f2_hsum(q)};
    row_sum<TPR, 1>(s, buf + W);
    rstd = rsqrtf(s[0] / p.D + p.eps);
    const f2 r = f2_all(rstd);
#pragma unroll
    for (int i = 0; i < EPT / 2; i++) v[i] = fmul2(v[i], r);
}

// Rows of more than one warp: a CTA walks rows, the next two on their way to shared memory
template <typename T, typename TR, int TPR, int EPT, int V>
struct NormRing {
    static constexpr int ROW = TPR * EPT, DEPTH = TPR > 32 && V == 4 ? 2 : 0;
    static constexpr int kGate = ROW * sizeof(T), kRes = 2 * kGate, kStage = kRes + ROW * sizeof(TR);
    static constexpr size_t bytes = (size_t)DEPTH * kStage;
};

template <typename T, typename TR, int TPR, int EPT, int V>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_fwd_kernel(NormParams p) {
    using Ring = NormRing<T, TR, TPR, EPT, V>;
    constexpr int DEPTH = Ring::DEPTH, RPC = TPR == 32 ? 4 : 1, P = EPT / 2;
    __shared__ float sums[TPR > 32 ? TPR / 32 * 8 : 1];
    extern __shared__ float4 norm_smem[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(norm_smem);
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x % TPR;
    const long long first = (long long)blockIdx.x * RPC + threadIdx.x / TPR, by = (long long)gridDim.x * RPC;
    RowAt here(first, DEPTH > 0 ? by : 0, p.L), ahead = here;        // without a ring every row has a warp or CTA of its own
    auto prefetch = [&](long long row, int stage) {
        if (row < p.rows) {
            auto at = [&](const Stream& s) { return ahead.of(s); };
            unsigned char* to = ring + stage * Ring::kStage;
            ring_issue<T, TPR, EPT>(to, static_cast<const T*>(p.x.p) + at(p.x), p.D, tid);
            if (p.gate.p) ring_issue<T, TPR, EPT>(to + Ring::kGate, static_cast<const T*>(p.gate.p) + at(p.gate), p.D, tid);
            if (p.res.p) ring_issue<TR, TPR, EPT>(to + Ring::kRes, static_cast<const TR*>(p.res.p) + at(p.res), p.D, tid);
        }
        cp_async_commit();
        ahead.next();
    };
    if constexpr (DEPTH > 0)
#pragma unroll
        for (int i = 0; i < DEPTH; i++) prefetch(first + i * by, i);
    int at_stage = 0;
    for (long long row = first; row < p.rows; row += by, here.next()) {
        float* buf = sums + (TPR > 32 ? at_stage * (TPR / 8) : 0);      // the rows' sums alternate between two sets of buffers
        auto at = [&](const Stream& s) { return here.of(s); };
        f2 x[P], r[P], g[P];
        if constexpr (DEPTH > 0) cp_async_wait<DEPTH - 1>();
        const unsigned char* stage = ring + at_stage * Ring::kStage;
        if constexpr (DEPTH > 0) {
            row_load<TPR, EPT, V>(reinterpret_cast<const T*>(stage), p.D, tid, x);
            if (p.res.p) row_load<TPR, EPT, V>(reinterpret_cast<const TR*>(stage + Ring::kRes), p.D, tid, r);
            if (p.gate.p) row_load<TPR, EPT, V>(reinterpret_cast<const T*>(stage + Ring::kGate), p.D, tid, g);
        } else {
            RawVec<T, V> rx[EPT / V], rg[EPT / V];
            RawVec<TR, V> rr[EPT / V];
            row_fetch<TPR, EPT, V>(static_cast<const T*>(p.x.p) + at(p.x), true, p.D, tid, rx);
            row_fetch<TPR, EPT, V>(static_cast<const TR*>(p.res.p) + at(p.res), p.res.p != nullptr, p.D, tid, rr);
            row_fetch<TPR, EPT, V>(static_cast<const T*>(p.gate.p) + at(p.gate), p.gate.p != nullptr, p.D, tid, rg);
            row_convert<EPT, V>(rx, x);
            row_convert<EPT, V>(rr, r);
            row_convert<EPT, V>(rg, g);
        }
        float stats[4] = {0.f, 1.f, 0.f, 1.f};
        if (p.pw) {
            row_normalise<TPR, EPT, V>(x, p, tid, buf, stats[0], stats[1]);
            f2 w[P], b[P];
            row_load<TPR, EPT, V>(p.pw, p.D, tid, w);
            if (p.pb) {
                row_load<TPR, EPT, V>(p.pb, p.D, tid, b);
#pragma unroll
                for (int i = 0; i < P; i++) x[i] = ffma2(x[i], w[i], b[i]);
            } else {
#pragma unroll
                for (int i = 0; i < P; i++) x[i] = fmul2(x[i], w[i]);
            }
        }
        if (p.gate.p) {
            gate_factor(p.act, g, g);
#pragma unroll
            for (int i = 0; i < P; i++) x[i] = fmul2(x[i], g[i]);
        }
        if (p.sv) row_load<TPR, EPT, V>(p.sv, p.D, tid, g);
        else
#pragma unroll
            for (int i = 0; i < P; i++) g[i] = f2_all(p.sval);
        if (p.res.p) {
#pragma unroll
            for (int i = 0; i < P; i++) x[i] = ffma2(x[i], g[i], r[i]);
        } else {
#pragma unroll
            for (int i = 0; i < P; i++) x[i] = fmul2(x[i], g[i]);
        }
        row_store<TPR, EPT, V>(static_cast<TR*>(p.r.p) + at(p.r), p.D, tid, x);
        row_normalise<TPR, EPT, V>(x, p, tid, buf + (TPR > 32 ? TPR / 16 : 0), stats[2], stats[3]);
        if constexpr (DEPTH > 0) prefetch(row + DEPTH * by, at_stage);      // every value of the stage has been used
        at_stage ^= 1;
        row_load<TPR, EPT, V>(p.w, p.D, tid, g);
        if (p.b) {
            row_load<TPR, EPT, V>(p.b, p.D, tid, r);
#pragma unroll
            for (int i = 0; i < P; i++) x[i] = ffma2(x[i], g[i], r[i]);
        } else {
#pragma unroll
            for (int i = 0; i < P; i++) x[i] = fmul2(x[i], g[i]);
        }
        row_store<TPR, EPT, V>(static_cast<T*>(p.y.p) + at(p.y), p.D, tid, x);
        if (p.stats && tid == 0) *reinterpret_cast<float4*>(p.stats + 4 * row) = make_float4(stats[0], stats[1], stats[2], stats[3]);
    }
}

template <typename T, typename TR, int TPR, int EPT>
static int norm_launch(const NormParams& p, bool vec, cudaStream_t st) {
    constexpr int RPC = TPR == 32 ? 4 : 1, threads = TPR == 32 ? 128 : TPR;
    long long ctas = ceil_div(p.rows, RPC);
    if (TPR > 32 && vec) {      // as many CTAs as stay resident: 16 warps and two rows of each are enough for the memory
        const long long most = (sm_count() > 0 ? sm_count() : 148) * (TPR == 128 ? (EPT == 8 ? 8LL : 4) : TPR == 256 ? 2 : 1);
        if (ctas > most) ctas = most;
    }
    if (ctas > 0x7fffffffLL) return FWP_ERR_SHAPE;
    if (vec) return launch_dependent_beside(norm_fwd_kernel<T, TR, TPR, EPT, 4>, p, dim3((unsigned)ctas), threads, NormRing<T, TR, TPR, EPT, 4>::bytes, st, "norm_fwd_kernel");
    return launch_dependent_beside(norm_fwd_kernel<T, TR, TPR, EPT, 1>, p, dim3((unsigned)ctas), threads, 0, st, "norm_fwd_kernel");
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
