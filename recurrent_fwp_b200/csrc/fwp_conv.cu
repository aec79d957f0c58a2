// Short causal convolution per channel (sm_100a), forward and backward.
//
//   p_t = bias + sum_j w_j x_{t-K+1+j},  out_t = p_t sigmoid(p_t)
//   gp_t = gout_t silu'(p_t),  gx_t = sum_j w_j gp_{t+K-1-j},  gw_j = sum_t gp_t x_{t-K+1+j}
//
// Bound by the bytes: forward one element in and one out per (n, t, d), backward two in and one out.  A warp owns 32 x V channels
// of one sequence and walks a span of steps with the last K - 1 inputs in registers, so every input is read once (and K - 1 of
// a neighbour's span, from L2); a block of four to eight rows is on its way while the one before it is worked on.  More rows in flight
// cost registers and with them warps: of 2 to 16 rows and 3 to 8 CTAs per SM these were the fastest (8 x 2048 x 2048, bf16, 4 taps: 31 us
// forward, 4.3 TB/s, and 55 us backward, 3.7 TB/s).  The backward walks forwards too: it forms p again from the inputs it needs
// for gw anyway, and gx K - 1 steps behind.
#include <type_traits>
#include "fwp_seq.cuh"

namespace fwp {

constexpr int kConvMaxK = 8;
constexpr int kConvWarps = 4;
constexpr int kConvSpan = 8;            // the shortest span: above K - 1, so that the first span alone sees the state

struct ConvParams {
    Stream x, state, out, gout, gx;     // state: rows are the K - 1 inputs before the first
    const float *w, *b;
    const int* lengths;
    float* part;                        // backward: [N * span groups][D * (K + 1)]
    int N, L, D, silu, span, spans;
};

// V neighbouring channels of a step: one float, or two pairs for the two-wide instructions
template <int V> struct Lanes;
template <> struct Lanes<1> {
    float v;
    __device__ __forceinline__ static Lanes all(float x) { return {x}; }
    __device__ __forceinline__ static Lanes of(const float (&x)[1]) { return {x[0]}; }
    __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = v; }
};
template <> struct Lanes<4> {
    f2 v[2];
    __device__ __forceinline__ static Lanes all(float x) { return {{f2_pack(x, x), f2_pack(x, x)}}; }
    __device__ __forceinline__ static Lanes of(const float (&x)[4]) { return {{f2_pack(x[0], x[1]), f2_pack(x[2], x[3])}}; }
    __device__ __forceinline__ void get(float (&x)[4]) const { f2_unpack(v[0], x[0], x[1]); f2_unpack(v[1], x[2], x[3]); }
};
__device__ __forceinline__ Lanes<1> fma_(Lanes<1> a, Lanes<1> b, Lanes<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Lanes<1> mul_(Lanes<1> a, Lanes<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Lanes<1> add_(Lanes<1> a, Lanes<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Lanes<4> fma_(Lanes<4> a, Lanes<4> b, Lanes<4> c) { return {{ffma2(a.v[0], b.v[0], c.v[0]), ffma2(a.v[1], b.v[1], c.v[1])}}; }
__device__ __forceinline__ Lanes<4> mul_(Lanes<4> a, Lanes<4> b) { return {{fmul2(a.v[0], b.v[0]), fmul2(a.v[1], b.v[1])}}; }
__device__ __forceinline__ Lanes<4> add_(Lanes<4> a, Lanes<4> b) { return {{fadd2(a.v[0], b.v[0]), fadd2(a.v[1], b.v[1])}}; }
template <int V>
__device__ __forceinline__ Lanes<V> sigmoid_(Lanes<V> a) {
    float e[V];
    mul_(a, Lanes<V>::all(-kLog2e)).get(e);
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = ex2_approx(e[i]);
    add_(Lanes<V>::of(e), Lanes<V>::all(1.f)).get(e);
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = rcp_approx(e[i]);
    return Lanes<V>::of(e);
}
template <typename T, int V>
__device__ __forceinline__ Lanes<V> lanes_of(const RawVec<T, V>& r) {
    float x[V];
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = r.get(i);
    return Lanes<V>::of(x);
}
template <int V, typename T>
__device__ __forceinline__ Lanes<V> load_lanes(const T* p) {
    float x[V];
    load_vec<V>(p, x);
    return Lanes<V>::of(x);
}

template <int K, int V>
__device__ __forceinline__ void conv_weights(const ConvParams& p, int d0, Lanes<V> (&w)[K], Lanes<V>& b) {
    float x[V];
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = p.b ? p.b[d0 + i] : 0.f;
    b = Lanes<V>::of(x);
#pragma unroll
    for (int j = 0; j < K; j++) {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = p.w[(long long)(d0 + i) * K + j];
        w[j] = Lanes<V>::of(x);
    }
}

// the K - 1 inputs before step t0 (steps below zero come from the state, or are zero)
template <typename T, int K, int V>
__device__ __forceinline__ void conv_window(const ConvParams& p, const T* x, int n, int t0, int d0, Lanes<V> (&win)[K]) {
#pragma unroll
    for (int j = 0; j < K - 1; j++) {
        const int t = t0 - (K - 1) + j;
        win[j] = Lanes<V>::all(0.f);
        if (t >= 0) win[j] = load_lanes<V>(x + t * p.x.sL);
        else if (p.state.p)
            win[j] = load_lanes<V>(static_cast<const float*>(p.state.p) + n * p.state.sN + (long long)(t + K - 1) * p.state.sL + d0);
    }
}

template <typename T, int K, int V>
__global__ void __launch_bounds__(kConvWarps * 32, K <= 4 ? 5 : 3) conv_fwd_kernel(ConvParams p) {
    constexpr int ROWS = V == 4 && sizeof(T) == 4 ? 4 : 8;           // rows loaded ahead of their use
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, n = blockIdx.z;
    const int d0 = (blockIdx.x * 32 + lane) * V;
    const int s = blockIdx.y * kConvWarps + (threadIdx.x >> 5);
    if (d0 >= p.D || s >= p.spans) return;
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
    const int t0 = s * p.span, t1 = min(t0 + p.span, len), tend = min(t0 + p.span, p.L);
    const T* x = static_cast<const T*>(p.x.p) + n * p.x.sN + d0;
    T* out = static_cast<T*>(p.out.p) + n * p.out.sN + d0;
    Lanes<V> w[K], b, win[K];
    if (t0 < t1 || s == 0) {
        conv_weights<K, V>(p, d0, w, b);
        conv_window<T, K, V>(p, x, n, t0, d0, win);
    }
    // the first span reads the state before the steps, and writes the one behind them: nobody else touches it
    if (s == 0 && p.state.p && K > 1) {
        float* st = static_cast<float*>(p.state.p) + n * p.state.sN + d0;
        float end[K][V];
#pragma unroll
        for (int j = 0; j < K - 1; j++) {
            // the inputs and the state before them are one sequence: K - 1 rows of state, then x; its rows from len on
            if (len + j >= K - 1) load_vec<V>(x + (len + j - (K - 1)) * p.x.sL, end[j]);
            else load_vec<V>(st + (len + j) * p.state.sL, end[j]);
        }
#pragma unroll
        for (int j = 0; j < K - 1; j++) store_vec<V>(st + j * p.state.sL, end[j]);
    }
    if (t0 < t1) {
        RawVec<T, V> raw[ROWS];        // rows behind the end repeat the last one
        auto fetch = [&](int t) {
#pragma unroll
            for (int r = 0; r < ROWS; r++) raw[r].load(x + min(t + r, t1 - 1) * p.x.sL);
        };
        fetch(t0);
        for (int t = t0; t < t1; t += ROWS) {
            RawVec<T, V> now[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r++) now[r] = raw[r];
            if (t + ROWS < t1) fetch(t + ROWS);
            T* to = out + t * p.out.sL;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                win[K - 1] = lanes_of(now[r]);
                Lanes<V> a = b;
#pragma unroll
                for (int j = 0; j < K; j++) a = fma_(w[j], win[j], a);
                if (p.silu) a = mul_(a, sigmoid_(a));
#pragma unroll
                for (int j = 0; j < K - 1; j++) win[j] = win[j + 1];
                float y[V];
                a.get(y);
                if (t + r < t1) store_vec<V>(to + r * p.out.sL, y);
            }
        }
    }
    const float zero[V] = {};
    for (int t = max(t0, t1); t < tend; t++) store_vec<V>(out + (long long)t * p.out.sL, zero);
}

template <typename T, int K, int V>
__global__ void __launch_bounds__(kConvWarps * 32, K > 4 ? 2 : sizeof(T) == 2 ? 4 : 3) conv_bwd_kernel(ConvParams p) {
    constexpr int ROWS = 4;
    __shared__ float red[kConvWarps][K + 1][32 * V];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.z;
    const int d0 = (blockIdx.x * 32 + lane) * V;
    const int s = blockIdx.y * kConvWarps + warp;
    const bool on = d0 < p.D && s < p.spans;
    const Lanes<V> none = Lanes<V>::all(0.f), one = Lanes<V>::all(1.f);
    Lanes<V> gw[K], gb = none;
#pragma unroll
    for (int j = 0; j < K; j++) gw[j] = none;
    if (on) {
        const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
        const int t0 = s * p.span, t1 = min(t0 + p.span, len), tend = min(t0 + p.span, p.L);
        const T* x = static_cast<const T*>(p.x.p) + n * p.x.sN + d0;
        const T* gout = static_cast<const T*>(p.gout.p) + n * p.gout.sN + d0;
        T* gx = static_cast<T*>(p.gx.p) + n * p.gx.sN + d0;
        if (t0 < t1) {
            Lanes<V> w[K], b, win[K], gp[K];               // gp[j]: of step u - K + 1 + j
            conv_weights<K, V>(p, d0, w, b);
            conv_window<T, K, V>(p, x, n, t0, d0, win);
#pragma unroll
            for (int j = 0; j < K; j++) gp[j] = none;
            const int uend = min(t1 + K - 1, len), ulast = uend - 1;     // steps from t1 on belong to the next span: only their gp counts here
            RawVec<T, V> rx[ROWS], rg[ROWS];
            auto fetch = [&](int u) {
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    rx[r].load(x + min(u + r, ulast) * p.x.sL);
                    rg[r].load(gout + min(u + r, ulast) * p.gout.sL);
                }
            };
            // ROWS steps from u0 on; INNER: all of them count in full, and so do the steps K - 1 before them
            auto block = [&](auto inner, int u0) {
                constexpr bool INNER = decltype(inner)::value;
                RawVec<T, V> nx[ROWS], ng[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; r++) { nx[r] = rx[r]; ng[r] = rg[r]; }
                if (u0 + ROWS < uend) fetch(u0 + ROWS);
                T* to = gx + (u0 - (K - 1)) * p.gx.sL;
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    const int u = u0 + r, t = u - (K - 1);
                    win[K - 1] = lanes_of(nx[r]);
                    Lanes<V> a = b, d = lanes_of(ng[r]);
#pragma unroll
                    for (int j = 0; j < K; j++) a = fma_(w[j], win[j], a);
                    if (p.silu) {
                        const Lanes<V> sg = sigmoid_(a);
                        // silu'(a) = sg (1 + a (1 - sg))
                        d = mul_(d, mul_(sg, fma_(a, fma_(sg, Lanes<V>::all(-1.f), one), one)));
                    }
                    if (!INNER && u >= uend) d = none;
                    gp[K - 1] = d;
                    if (INNER || u < t1) {
                        gb = add_(gb, d);
#pragma unroll
                        for (int j = 0; j < K; j++) gw[j] = fma_(d, win[j], gw[j]);
                    }
                    Lanes<V> q = mul_(w[0], gp[K - 1]);
#pragma unroll
                    for (int j = 1; j < K; j++) q = fma_(w[j], gp[K - 1 - j], q);       // gp of step t + K - 1 - j
#pragma unroll
                    for (int j = 0; j < K - 1; j++) { win[j] = win[j + 1]; gp[j] = gp[j + 1]; }
                    float g[V];
                    q.get(g);
                    if (INNER || (t >= t0 && t < t1)) store_vec<V>(to + r * p.gx.sL, g);
                }
            };
            fetch(t0);
            for (int u0 = t0; u0 < t1 + K - 1; u0 += ROWS) {
                if (u0 - (K - 1) >= t0 && u0 + ROWS <= t1) block(std::true_type(), u0);
                else block(std::false_type(), u0);
            }
        }
        const float zero[V] = {};
        for (int t = max(t0, t1); t < tend; t++) store_vec<V>(gx + (long long)t * p.gx.sL, zero);
    }
    float v[V];
    gb.get(v);
#pragma unroll
    for (int i = 0; i < V; i++) red[warp][K][lane * V + i] = v[i];
#pragma unroll
    for (int j = 0; j < K; j++) {
        gw[j].get(v);
#pragma unroll
        for (int i = 0; i < V; i++) red[warp][j][lane * V + i] = v[i];
    }
    __syncthreads();
    // partial sums of the CTA: weights as [D][K], then the bias
    float* part = p.part + ((long long)n * gridDim.y + blockIdx.y) * p.D * (K + 1);
    for (int i = threadIdx.x; i < 32 * V * (K + 1); i += kConvWarps * 32) {
        const int j = i / (32 * V), c = i - j * (32 * V), d = blockIdx.x * 32 * V + c;
        if (d >= p.D) continue;
        float a = 0.f;
#pragma unroll
        for (int q = 0; q < kConvWarps; q++) a += red[q][j][c];
        part[j == K ? (long long)p.D * K + d : (long long)d * K + j] = a;
    }
}

static long long conv_sms() { return sm_count() > 0 ? sm_count() : 148; }
// Steps a warp walks: long spans read fewer neighbours' steps, short ones fill the machine when there are few channels.
static int conv_span(int N, int L, int D, int V, long long sms) {
    const long long columns = (long long)N * ceil_div(D, 32 * V);
    int span = 64;
    while (span > kConvSpan && columns * ceil_div(L, span) < sms * 16) span >>= 1;
    while (ceil_div(L, (long long)span * kConvWarps) > 65535) span <<= 1;      // the grid's limit
    return span;
}

static int conv_check(int N, int L, int D, int K, const fwp_tensor* x, const float* w, const float* b, const fwp_tensor* state,
                      const int* lengths, int io_dtype) {
    if (N < 0 || L < 0 || D < 0 || K < 1) return FWP_ERR_SHAPE;
    if (io_dtype != FWP_F32 && io_dtype != FWP_BF16) return FWP_ERR_DTYPE;
    if (K > kConvMaxK) return FWP_ERR_UNSUPPORTED;
    if (N > 65535 || L > kMaxSteps) return FWP_ERR_SHAPE;
    if (D && !w) return FWP_ERR_NULL;
    if (!aligned4(w) || !aligned4(b) || !aligned4(lengths)) return FWP_ERR_ALIGN;
    if (!N || !L || !D) return FWP_OK;
    if (int rc = check_tensor(x, io_dtype == FWP_F32 ? 4 : 2, true)) return rc;
    return check_tensor(state, 4, false);
}

static bool conv_vectors(const ConvParams& p, int esz) {
    return p.D % 4 == 0 && rows_aligned(p.x, esz, 4 * esz) && rows_aligned(p.state, 4, 16) && rows_aligned(p.out, esz, 4 * esz) &&
           rows_aligned(p.gout, esz, 4 * esz) && rows_aligned(p.gx, esz, 4 * esz);
}

template <typename T, int K, int V>
static int conv_launch(ConvParams p, bool backward, cudaStream_t st) {
    p.span = conv_span(p.N, p.L, p.D, V, conv_sms());
    p.spans = (int)ceil_div(p.L, p.span);
    const dim3 grid((unsigned)ceil_div(p.D, 32 * V), (unsigned)ceil_div(p.spans, kConvWarps), (unsigned)p.N);
    if (backward) return launch_dependent(conv_bwd_kernel<T, K, V>, p, grid, kConvWarps * 32, 0, st, "conv_bwd_kernel");
    return launch_dependent(conv_fwd_kernel<T, K, V>, p, grid, kConvWarps * 32, 0, st, "conv_fwd_kernel");
}
template <typename T, int V>
static int conv_taps(int K, const ConvParams& p, bool backward, cudaStream_t st) {
    switch (K) {
        case 1: return conv_launch<T, 1, V>(p, backward, st);
        case 2: return conv_launch<T, 2, V>(p, backward, st);
        case 3: return conv_launch<T, 3, V>(p, backward, st);
        case 4: return conv_launch<T, 4, V>(p, backward, st);
        case 5: return conv_launch<T, 5, V>(p, backward, st);
        case 6: return conv_launch<T, 6, V>(p, backward, st);
        case 7: return conv_launch<T, 7, V>(p, backward, st);
    }
    return conv_launch<T, 8, V>(p, backward, st);
}
static int conv_dispatch(int K, const ConvParams& p, bool backward, int io_dtype, cudaStream_t st) {
    if (io_dtype == FWP_F32) return conv_vectors(p, 4) ? conv_taps<float, 4>(K, p, backward, st) : conv_taps<float, 1>(K, p, backward, st);
    return conv_vectors(p, 2) ? conv_taps<__nv_bfloat16, 4>(K, p, backward, st) : conv_taps<__nv_bfloat16, 1>(K, p, backward, st);
}

// rows of partial sums: at most those of the narrowest form
static long long conv_part_rows(int N, int L, int D, long long sms) {
    long long most = 0;
    for (int V : {1, 4}) {
        int span = conv_span(N, L, D, V, sms);
        const long long rows = (long long)N * ceil_div(ceil_div(L, span), kConvWarps);
        most = rows > most ? rows : most;
    }
    return most;
}

// ---------------------------------------------------------------- sums of partial gradients
// 32 columns per CTA, its other threads down the rows: a column of partial sums is as long as the kernel before it had CTAs.  Few columns take
// 32 rows at a time (592 x 512: 5.6 us, 6.5 with eight), many eight (296 x 20480: 9.7 us, 17.6 with 32: waves of CTAs)
template <int ROWS>
__global__ void __launch_bounds__(ROWS * 32) column_sums_kernel(ColumnSums p) {
    __shared__ float red[ROWS][33];
    griddep_wait();
    griddep_launch_dependents();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * 32 + tx;
    float a = 0.f;
    if (c < p.W)
#pragma unroll 4
        for (int r = ty; r < p.P; r += ROWS) a += p.part[r * p.W + c];
    red[ty][tx] = a;
    __syncthreads();
    if (ty || c >= p.W) return;
#pragma unroll
    for (int i = 1; i < ROWS; i++) a += red[i][tx];
    long long from = 0;
#pragma unroll
    for (int k = 0; k < kSumSegments; k++) {
        if (c >= from && c < p.end[k]) {
            if (p.out[k]) p.out[k][c - from] = a;
            return;
        }
        from = p.end[k];
    }
}

int launch_column_sums(const ColumnSums& p, cudaStream_t st) {
    const dim3 grid((unsigned)ceil_div(p.W, 32));
    if (p.P > 32 && p.W < 32 * 256) return launch_dependent(column_sums_kernel<32>, p, grid, 1024, 0, st, nullptr);
    return launch_dependent(column_sums_kernel<8>, p, grid, 256, 0, st, nullptr);
}

}  // namespace fwp

using namespace fwp;

FWP_API int fwp_causal_conv_forward(int N, int L, int D, int K, const fwp_tensor* x, const float* weight, const float* bias,
                                    const fwp_tensor* state, const int* lengths, const fwp_tensor* out, int silu, int io_dtype,
                                    void* stream, int device) {
    int rc;
    if ((rc = conv_check(N, L, D, K, x, weight, bias, state, lengths, io_dtype)) || !N || !L || !D) return rc;
    if ((rc = check_tensor(out, io_dtype == FWP_F32 ? 4 : 2, true))) return rc;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    ConvParams p = {stream_of(x), stream_of(state), stream_of(out), {}, {}, weight, bias, lengths, nullptr, N, L, D, silu ? 1 : 0, 0, 0};
    return conv_dispatch(K, p, false, io_dtype, (cudaStream_t)stream);
}

FWP_API int64_t fwp_causal_conv_backward_scratch_floats(int N, int L, int D, int K) {
    if (N <= 0 || L <= 0 || D <= 0 || K < 1 || K > kConvMaxK) return 0;
    return conv_part_rows(N, L, D, most_sms()) * D * (K + 1);        // more SMs never take fewer rows
}

FWP_API int fwp_causal_conv_backward(int N, int L, int D, int K, const fwp_tensor* x, const float* weight, const float* bias,
                                     const fwp_tensor* start, const int* lengths, const fwp_tensor* grad_out, const fwp_tensor* grad_x,
                                     float* grad_weight, float* grad_bias, float* scratch, int64_t scratch_floats, int silu,
                                     int io_dtype, void* stream, int device) {
    const int esz = io_dtype == FWP_F32 ? 4 : 2;
    int rc;
    if ((rc = conv_check(N, L, D, K, x, weight, bias, start, lengths, io_dtype))) return rc;
    if (N && L && D && ((rc = check_tensor(grad_out, esz, true)) || (rc = check_tensor(grad_x, esz, true)))) return rc;
    if (D && !grad_weight) return FWP_ERR_NULL;
    if (!aligned4(grad_weight) || !aligned4(grad_bias)) return FWP_ERR_ALIGN;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    cudaStream_t st = (cudaStream_t)stream;
    if (!N || !L || !D) {               // no steps: sums of nothing
        cudaError_t e = D ? cudaMemsetAsync(grad_weight, 0, sizeof(float) * D * K, st) : cudaSuccess;
        if (e == cudaSuccess && D && grad_bias) e = cudaMemsetAsync(grad_bias, 0, sizeof(float) * D, st);
        return e == cudaSuccess ? FWP_OK : set_cuda_error(e);
    }
    if (!scratch || !aligned16(scratch) || scratch_floats < conv_part_rows(N, L, D, conv_sms()) * D * (K + 1)) return FWP_ERR_SCRATCH;
    ConvParams p = {stream_of(x), stream_of(start), {}, stream_of(grad_out), stream_of(grad_x), weight, bias, lengths, scratch,
                    N, L, D, silu ? 1 : 0, 0, 0};
    if ((rc = conv_dispatch(K, p, true, io_dtype, st))) return rc;
    const int V = conv_vectors(p, esz) ? 4 : 1;
    const int span = conv_span(N, L, D, V, conv_sms());
    const long long dk = (long long)D * K;
    ColumnSums s = {scratch, (int)(N * ceil_div(ceil_div(L, span), kConvWarps)), dk + D, {grad_weight, grad_bias}, {dk, dk + D}};
    return launch_column_sums(s, st);
}
