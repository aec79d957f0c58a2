// The norm behind a block, its gate and residual scale, the residual sum and the norm before the next block, in one pass each way:
//
//   t = norm(x; pw, pb) or x,  u = t act(gate) or t,  r = residual + s u,  y = norm(r; w, b)
//
// Bound by the bytes: every row is held in the registers of the threads that own it (one warp up to 512 elements in the forward and 256 in
// the plain backward, several warps beyond), so each stream moves once: 16384 rows of 4096, all parts, bf16 with an fp32 residual, 178 us forward
// (5.3 TB/s) and 363 us backward (4.1 TB/s, one CTA of 255 registers per SM).  With the residual sum alone, rows of 256 to 8192: 88 to 104 % of the
// copy rate forward and 87 to 98 % backward beside an fp32 residual, 71 to 83 % and 71 to 80 % where all streams are bf16.  Means and variances are taken in fp32 over the unrounded values, the
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

// Sequence and step of a row, carried from row to row: a 64-bit division per row is as many instructions as the row's arithmetic.
struct RowAt {
    long long n, by_n;
    int l, by_l, L;
    __device__ __forceinline__ RowAt(long long row, long long by, int L_) : L(L_) {
        if ((row | by) >> 32) {
            n = row / L; l = (int)(row - n * L);
            by_n = by / L; by_l = (int)(by - by_n * L);
        } else {
            const unsigned q = (unsigned)row / (unsigned)L, b = (unsigned)by / (unsigned)L;
            n = q; l = (int)((unsigned)row - q * (unsigned)L);
            by_n = b; by_l = (int)((unsigned)by - b * (unsigned)L);
        }
    }
    __device__ __forceinline__ void next() {
        n += by_n;
        l += by_l;
        if (l >= L || l < 0) { l -= L; n++; }       // below zero: the sum passed 2^31
    }
    __device__ __forceinline__ long long of(const Stream& s) const { return n * s.sN + l * s.sL; }
};

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

// a thread's elements of a row, pieces of V that are TPR pieces apart, in pairs for the two-wide instructions; zero beyond the row
template <int TPR, int EPT, int V, typename T>
__device__ __forceinline__ void row_load(const T* p, int D, int tid, f2 (&v)[EPT / 2]) {
    if constexpr (V == 4) {
#pragma unroll
        for (int k = 0; k < EPT / 4; k++) {
            const int at = (k * TPR + tid) * 4;
            float q[4] = {};
            if (at < D) load_vec<4>(p + at, q);
            v[2 * k] = f2_pack(q[0], q[1]);
            v[2 * k + 1] = f2_pack(q[2], q[3]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < EPT / 2; k++) {
            const int at = 2 * k * TPR + tid;
            v[k] = f2_pack(at < D ? to_f32(p[at]) : 0.f, at + TPR < D ? to_f32(p[at + TPR]) : 0.f);
        }
    }
}
// the same in two steps, so that the loads of several streams are under way before the first is converted
template <int TPR, int EPT, int V, typename T>
__device__ __forceinline__ void row_fetch(const T* p, bool on, int D, int tid, RawVec<T, V> (&raw)[EPT / V]) {
#pragma unroll
    for (int k = 0; k < EPT / V; k++) {
        const int at = (k * TPR + tid) * V;
        raw[k].clear();
        if (on && at < D) raw[k].load(p + at);
    }
}
template <int EPT, int V, typename T>
__device__ __forceinline__ void row_convert(const RawVec<T, V> (&raw)[EPT / V], f2 (&v)[EPT / 2]) {
#pragma unroll
    for (int i = 0; i < EPT / 2; i++) v[i] = f2_pack(raw[2 * i / V].get(2 * i % V), raw[(2 * i + 1) / V].get((2 * i + 1) % V));
}
template <int TPR, int EPT, int V, typename T>
__device__ __forceinline__ void row_store(T* p, int D, int tid, const f2 (&v)[EPT / 2]) {
    if constexpr (V == 4) {
#pragma unroll
        for (int k = 0; k < EPT / 4; k++) {
            const int at = (k * TPR + tid) * 4;
            float q[4];
            f2_unpack(v[2 * k], q[0], q[1]);
            f2_unpack(v[2 * k + 1], q[2], q[3]);
            if (at < D) store_vec<4>(p + at, q);
        }
    } else {
#pragma unroll
        for (int k = 0; k < EPT / 2; k++) {
            const int at = 2 * k * TPR + tid;
            float lo, hi;
            f2_unpack(v[k], lo, hi);
            if (at < D) p[at] = from_f32<T>(lo);
            if (at + TPR < D) p[at + TPR] = from_f32<T>(hi);
        }
    }
}
// v with zeros beyond the row, where a mean has been taken off
template <int TPR, int EPT, int V>
__device__ __forceinline__ void row_cut(int D, int tid, f2 (&v)[EPT / 2]) {
    if (D == TPR * EPT) return;
#pragma unroll
    for (int k = 0; k < EPT / 2; k++) {
        if constexpr (V == 4) {
            v[k] = ((k / 2) * TPR + tid) * 4 < D ? v[k] : 0;
        } else {
            float lo, hi;
            f2_unpack(v[k], lo, hi);
            const int at = 2 * k * TPR + tid;
            v[k] = f2_pack(at < D ? lo : 0.f, at + TPR < D ? hi : 0.f);
        }
    }
}
__device__ __forceinline__ f2 f2_all(float x) { return f2_pack(x, x); }
__device__ __forceinline__ f2 sigmoid2(f2 x) {
    float lo, hi;
    f2_unpack(fmul2(x, f2_all(-kLog2e)), lo, hi);
    f2_unpack(fadd2(f2_pack(ex2_approx(lo), ex2_approx(hi)), f2_all(1.f)), lo, hi);
    return f2_pack(rcp_approx(lo), rcp_approx(hi));
}
// the gate's factor
template <int n>
__device__ __forceinline__ void gate_factor(int act, const f2 (&g)[n], f2 (&a)[n]) {
    if (act == 2) {
#pragma unroll
        for (int i = 0; i < n; i++) a[i] = g[i];
    } else {
#pragma unroll
        for (int i = 0; i < n; i++) {
            const f2 s = sigmoid2(g[i]);
            a[i] = act == 1 ? s : fmul2(g[i], s);
        }
    }
}
// the factor, and its derivative in place of the gate
template <int n>
__device__ __forceinline__ void gate_factor_and_grad(int act, f2 (&g)[n], f2 (&a)[n]) {
    const f2 one = f2_all(1.f), minus = f2_all(-1.f);
    if (act == 2) {
#pragma unroll
        for (int i = 0; i < n; i++) { a[i] = g[i]; g[i] = one; }
    } else if (act == 1) {
#pragma unroll
        for (int i = 0; i < n; i++) {
            a[i] = sigmoid2(g[i]);
            g[i] = fmul2(a[i], ffma2(a[i], minus, one));
        }
    } else {
#pragma unroll
        for (int i = 0; i < n; i++) {
            const f2 s = sigmoid2(g[i]), q = ffma2(s, minus, one);
            a[i] = fmul2(g[i], s);
            g[i] = fmul2(s, ffma2(g[i], q, one));
        }
    }
}

// The next rows of a thread's streams on their way to shared memory: every thread copies and reads back its own pieces, so the ring needs no
// barrier.  A row's copy into a stage is issued once the values that were in it have been used.
template <typename T, int TPR, int EPT>
__device__ __forceinline__ void ring_issue(unsigned char* stage, const T* row, int D, int tid) {
#pragma unroll
    for (int k = 0; k < EPT / 4; k++) {
        const int at = (k * TPR + tid) * 4;
        if (at >= D) continue;
        if constexpr (sizeof(T) == 4) cp_async16(stage + at * 4, row + at);
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(stage + at * 2)), "l"(row + at) : "memory");
    }
}

#endif
}  // namespace fwp
