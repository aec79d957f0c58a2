// The norm behind a block, its gate and residual scale, the residual sum and the norm before the next block, in one pass each way:
//
//   t = norm(x; pw, pb) or x,  u = t act(gate) or t,  r = residual + s u,  y = norm(r; w, b)
//
// Bound by the bytes: every row is held in the registers of the threads that own it (one warp up to 1024 elements in the forward and 256 in
// the backward, several warps beyond), so each stream moves once.  Means and variances are taken in fp32 over the unrounded values, the
// variance around the mean.  The backward forms r again from the forward's inputs: r itself is rounded where it is stored in bf16, which
// would cost the fp32 gradients of the weights their accuracy (1e-3 against 1e-6).
#pragma once
#include "fwp_seq.cuh"

namespace fwp {

constexpr int kNormMaxD = 8192;

struct NormParams {
    Stream x, res, gate, y, r;
    Stream gy, gr, gx, gres, ggate;
    const float *sv, *pw, *pb, *w, *b;
    float sval, eps;
    float* stats;               // per row: mean and 1 / sd of the norm behind the block, of the norm before the next
    float* part;
    int L, D, rms, act;
    long long rows;
};

static inline int norm_check(int N, int L, int D, const fwp_tensor* x, const fwp_tensor* residual, const fwp_tensor* gate, const float* sv,
                             const float* pw, const float* pb, const float* w, const float* b, int gate_act, int io, int rio) {
    if (N < 0 || L < 0 || D < 0) return FWP_ERR_SHAPE;
    if ((io != FWP_F32 && io != FWP_BF16) || (rio != io && rio != FWP_F32)) return FWP_ERR_DTYPE;
    if (D > kNormMaxD || gate_act < 0 || gate_act > 2) return FWP_ERR_UNSUPPORTED;
    if (D && !w) return FWP_ERR_NULL;
    for (const float* q : {sv, pw, pb, w, b})
        if (!aligned4(q)) return FWP_ERR_ALIGN;
    if (!N || !L || !D) return FWP_OK;
    const int esz = io == FWP_F32 ? 4 : 2;
    int rc;
    if ((rc = check_tensor(x, esz, true)) || (rc = check_tensor(residual, rio == FWP_F32 ? 4 : 2, false)) || (rc = check_tensor(gate, esz, false)))
        return rc;
    return FWP_OK;
}

static inline NormParams norm_params(int N, int L, int D, const fwp_tensor* x, const fwp_tensor* residual, const fwp_tensor* gate,
                                     const float* sv, float sval, const float* pw, const float* pb, const float* w, const float* b,
                                     int rms, int gate_act) {
    NormParams p = {};
    p.x = stream_of(x); p.res = stream_of(residual); p.gate = stream_of(gate);
    p.sv = sv; p.pw = pw; p.pb = pb; p.w = w; p.b = b;
    p.sval = sval;
    p.L = L; p.D = D; p.rms = rms ? 1 : 0; p.act = gate_act;
    p.rows = (long long)N * L;
    return p;
}
static inline bool norm_vectors(const NormParams& p) {
    bool ok = p.D % 4 == 0;
    for (const float* q : {p.sv, p.pw, p.pb, p.w, p.b}) ok = ok && aligned16(q);
    return ok;
}

#ifdef __CUDACC__

// sums over the TPR threads of a row; one barrier, the caller alternates `buf`
template <int TPR, int n>
__device__ __forceinline__ void row_sum(float (&v)[n], float* buf) {
#pragma unroll
    for (int i = 0; i < n; i++)
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < n; i++) buf[i * W + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < n; i++) {
            float a = lane < W ? buf[i * W + lane] : 0.f;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            v[i] = a;
        }
    }
}

// a thread's elements of a row: pieces of V, TPR pieces apart
template <int TPR, int EPT, int V, typename T>
__device__ __forceinline__ void row_load(const T* p, int D, int tid, float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < EPT / V; k++) {
        const int at = (k * TPR + tid) * V;
        float q[V] = {};
        if (at < D) load_vec<V>(p + at, q);
#pragma unroll
        for (int i = 0; i < V; i++) v[k * V + i] = q[i];
    }
}
template <int TPR, int EPT, int V, typename T>
__device__ __forceinline__ void row_store(T* p, int D, int tid, const float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < EPT / V; k++) {
        const int at = (k * TPR + tid) * V;
        float q[V];
#pragma unroll
        for (int i = 0; i < V; i++) q[i] = v[k * V + i];
        if (at < D) store_vec<V>(p + at, q);
    }
}
template <int TPR, int V>
__device__ __forceinline__ bool row_has(int i, int D, int tid) { return ((i / V) * TPR + tid) * V < D; }

__device__ __forceinline__ float gate_of(int act, float g) { return act == 2 ? g : act == 1 ? sigmoidf_(g) : g * sigmoidf_(g); }
__device__ __forceinline__ float gate_grad_of(int act, float g) {
    const float s = sigmoidf_(g);
    return act == 2 ? 1.f : act == 1 ? s * (1.f - s) : silu_grad_of(g, s);
}

#endif
}  // namespace fwp
