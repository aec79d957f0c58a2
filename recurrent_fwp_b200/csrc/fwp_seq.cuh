// What the operators of a state-space layer share (fwp_conv.cu, fwp_scan.cu, fwp_norm*.cu): (N, L, D) streams, vector
// accesses, sums over lanes, and the sum of per-CTA partial gradients in a fixed order.
#pragma once
#include "fwp_core.cuh"

namespace fwp {

struct Stream {          // an (N, L, D) tensor with unit inner stride
    void* p;
    long long sN, sL;
};
static inline Stream stream_of(const fwp_tensor* t) {
    Stream s = {nullptr, 0, 0};
    if (t && t->data) { s.p = t->data; s.sN = t->stride[0]; s.sL = t->stride[2]; }
    return s;
}
static inline bool given(const fwp_tensor* t) { return t && t->data; }

// rows of the stream can be moved in pieces of `bytes` bytes
static inline bool rows_aligned(const Stream& s, int esz, int bytes) {
    return !s.p || ((reinterpret_cast<uintptr_t>(s.p) % bytes) == 0 && (s.sN * esz) % bytes == 0 && (s.sL * esz) % bytes == 0);
}
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

constexpr int kMaxSteps = 0x7fff0000;       // of a sequence: the step behind a span's end is an int

static inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Sums over the rows of part[P][W], columns cut into segments that go to tensors of their own (null: not wanted).  The order of
// addition depends on P alone.
constexpr int kSumSegments = 5;
struct ColumnSums {
    const float* part;
    int P;
    long long W;
    float* out[kSumSegments];
    long long end[kSumSegments];       // first column behind each segment
};
int launch_column_sums(const ColumnSums& p, cudaStream_t st);

// launch_dependent for kernels with static shared memory beside the dynamic: the two together may pass 48 KB
template <typename K, typename P>
static int launch_dependent_beside(K kern, const P& p, dim3 grid, int threads, size_t bytes, cudaStream_t st, const char* name) {
    if (bytes > 32 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return set_cuda_error(e);
    }
    return launch_dependent(kern, p, grid, threads, bytes, st, name);
}

#ifdef __CUDACC__

__device__ __forceinline__ f2 fmul2(f2 a, f2 b) {
    f2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// V consecutive elements as floats; V = 4 needs an address aligned to 4 elements
template <int V>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[V]) {
    if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
        v[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[V]) {
    if constexpr (V == 4) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
    } else {
        v[0] = to_f32(*p);
    }
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *p = v[0];
}
template <int V>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[V]) {
    if constexpr (V == 4) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        uint2 t;
        t.x = *reinterpret_cast<unsigned*>(&a);
        t.y = *reinterpret_cast<unsigned*>(&b);
        *reinterpret_cast<uint2*>(p) = t;
    } else {
        *p = from_f32<__nv_bfloat16>(v[0]);
    }
}

// V elements as they are in memory, converted where they are used: a conversion next to the load would wait for it
template <typename T, int V> struct RawVec;
template <typename T> struct RawVec<T, 1> {
    T v;
    __device__ __forceinline__ void clear() { v = from_f32<T>(0.f); }
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ float get(int) const { return to_f32(v); }
};
template <> struct RawVec<float, 4> {
    float4 v;
    __device__ __forceinline__ void clear() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ float get(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
};
template <> struct RawVec<__nv_bfloat16, 4> {
    uint2 v;
    __device__ __forceinline__ void clear() { v = make_uint2(0u, 0u); }
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ float get(int i) const {
        const unsigned w = i < 2 ? v.x : v.y;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
};

// Sums of `n` values over LANES lanes that are STRIDE apart.  While there are more values than one the halves of the lanes take half of
// the values each (n / 2 shuffles), afterwards plain butterflies.  Where n >= LANES a lane ends with n / LANES values: those whose index
// is i * LANES... in the order of bits: the lane with index l = (lane / STRIDE) % LANES holds values l * (n / LANES) ... + n / LANES - 1
// in v[0 ...]; where n < LANES it holds value l / (LANES / n) in v[0].
template <int n, int LANES, int STRIDE>
__device__ __forceinline__ void sum_lanes(float (&v)[n], int lane) {
    constexpr unsigned kAll = 0xffffffffu;
    int left = n;
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1) {
        if (left > 1) {
            const bool hi = lane & (o * STRIDE);
            left >>= 1;
#pragma unroll
            for (int i = 0; i < n / 2; i++)
                if (i < left) {
                    const float keep = hi ? v[i + left] : v[i], send = hi ? v[i] : v[i + left];
                    v[i] = keep + __shfl_xor_sync(kAll, send, o * STRIDE);
                }
        } else {
            v[0] += __shfl_xor_sync(kAll, v[0], o * STRIDE);
        }
    }
}

// sigmoid(x) and x sigmoid(x) with its derivative; a few ulp, 0 and 1 at the ends, NaN for NaN
__device__ __forceinline__ float silu_of(float x, float sig) { return x * sig; }
__device__ __forceinline__ float silu_grad_of(float x, float sig) { return sig * (1.f + x * (1.f - sig)); }

#endif
}  // namespace fwp
