// Parameters and device pieces of the selective scan, shared by its forward (fwp_scan.cu) and backward (fwp_scan_bwd.cu).
#pragma once
#include <cfloat>
#include "fwp_seq.cuh"

namespace fwp {

constexpr int kScanMaxS = 64;
// The forward of a call with a backward keeps the state before every eighth step: 8 bytes per (step, channel) each way at S = 16, beside
// about 8 and 14 of streams in bf16.  The backward holds half a tile's states and decays in registers and forms the first half's twice; from
// states kept farther apart it would form all of them once more.
constexpr int kScanKeep = 8;

struct ScanParams {
    Stream x, dt, z, out;
    Row4 B, C;              // (N, G, L, S)
    const float *A, *skip, *dt_bias;
    const int* lengths;
    float* state;           // (N, D, S), null: zeros
    long long state_sN, state_sD;
    bool state_vec;         // a single step moves rows of the state, of B and of C in pieces of four
    bool pairs;             // the rows of two neighbouring channels move as one
    float* checkpoints;     // [N][ceil(L / 8)][D][scan_row(S)]
    float *ends, *dsums;    // [N][spans][D][S] and [N][spans][D]
    int N, L, D, S, G, softplus, span, spans;
    // backward
    Stream gout, gx, gdt, gz;
    float *bc, *sums;       // partial gradients of B and C, and of A, skip and dt_bias
    Row4 gBr, gCr;
};

// what a pass over the spans of time is for
enum ScanPass { SCAN_WHOLE = 0, SCAN_ENDS = 1 };

// joins what a pass over the spans left in ends and dsums into the spans' starts; `backwards`: from the last span, which starts from zero
int launch_scan_join(const ScanParams& p, bool backwards, cudaStream_t st);

// lanes that hold the states of one channel, four each
static inline int scan_lanes(int S) { return S <= 4 ? 1 : S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }
#ifdef __CUDACC__
__host__ __device__
#endif
static inline int scan_row(int S) { return (S + 3) & ~3; }

static inline int scan_check(int N, int L, int D, int S, int G, const fwp_tensor* x, const fwp_tensor* dt, const float* A,
                             const fwp_tensor* B, const fwp_tensor* C, const float* skip, const fwp_tensor* z, const float* dt_bias,
                             const int* lengths, int io_dtype) {
    if (N < 0 || L < 0 || D < 0 || S < 1 || G < 1 || D % G || N > 65535 || L > kMaxSteps) return FWP_ERR_SHAPE;
    if (io_dtype != FWP_F32 && io_dtype != FWP_BF16) return FWP_ERR_DTYPE;
    if (S > kScanMaxS) return FWP_ERR_UNSUPPORTED;
    if (D && !A) return FWP_ERR_NULL;
    if (!aligned4(A) || !aligned4(skip) || !aligned4(dt_bias) || !aligned4(lengths)) return FWP_ERR_ALIGN;
    if (!N || !L || !D) return FWP_OK;
    const int esz = io_dtype == FWP_F32 ? 4 : 2;
    int rc;
    if ((rc = check_tensor(x, esz, true)) || (rc = check_tensor(dt, esz, true)) || (rc = check_tensor(B, esz, true)) ||
        (rc = check_tensor(C, esz, true)) || (rc = check_tensor(z, esz, false)))
        return rc;
    return FWP_OK;
}

static inline ScanParams scan_params(int N, int L, int D, int S, int G, const fwp_tensor* x, const fwp_tensor* dt, const float* A,
                                     const fwp_tensor* B, const fwp_tensor* C, const float* skip, const fwp_tensor* z,
                                     const float* dt_bias, const int* lengths, int softplus) {
    ScanParams p = {};
    p.x = stream_of(x); p.dt = stream_of(dt); p.z = stream_of(z);
    p.B = row4(B); p.C = row4(C);
    p.A = A; p.skip = skip; p.dt_bias = dt_bias; p.lengths = lengths;
    p.N = N; p.L = L; p.D = D; p.S = S; p.G = G; p.softplus = softplus ? 1 : 0;
    return p;
}

#ifdef __CUDACC__

// log(1 + e^x).  With e = e^-|x|: max(x, 0) + log(1 + e), and log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3, by its power series to s^15 (the
// next term is below 1e-9).  Relative error 3e-7 + 7e-8 |x| for negative x, where the rounded product in the exponential's argument is all that
// counts (measured 9e-7 at -20, 3.9e-6 at -87), and zero below -87.3, where e^x leaves the normal floats; 1e-7 for x > 1.
__device__ __forceinline__ float softplus_(float x) {
    const float e = ex2_approx(-fabsf(x) * kLog2e), s = e * rcp_approx(2.f + e), q = s * s;
    float r = 1.f / 15.f;
    r = fmaf(r, q, 1.f / 13.f);
    r = fmaf(r, q, 1.f / 11.f);
    r = fmaf(r, q, 1.f / 9.f);
    r = fmaf(r, q, 1.f / 7.f);
    r = fmaf(r, q, 1.f / 5.f);
    r = fmaf(r, q, 1.f / 3.f);
    r = fmaf(r, q, 1.f);
    return fmaf(2.f * s, r, fmaxf(x, 0.f));     // a NaN is in s
}

// A log2(e).  Minus infinity, a state that keeps nothing, counts as the most negative float: steps of size zero, those behind the end of a
// sequence among them, leave such a state alone too, where zero times infinity would be NaN.
__device__ __forceinline__ float rate_of(float a) {
    a *= kLog2e;
    return a < -FLT_MAX ? -FLT_MAX : a;
}

// exp(delta A) from A log2(e).  A slow channel multiplies a thousand of these, so it is the mean error of the exponential instruction that
// its state shows: measured -19e-9 (relative) for arguments between -0.1 and -0.002, -5e-9 below.  2^-26 on the argument, which rides on the
// product for free, makes that -9e-9 and +5e-9; zero still gives exactly one.  The gradient of A over 2048 steps: 1.6e-6 -> 0.7e-6 off.
constexpr float kDecayCentre = 1.f / 67108864.f;
__device__ __forceinline__ float decay_of(float delta, float a) { return ex2_approx(fmaf(delta, a, kDecayCentre)); }
__device__ __forceinline__ f2 decay_pair(f2 delta, f2 a) {
    float lo, hi;
    f2_unpack(ffma2(delta, a, f2_pack(kDecayCentre, kDecayCentre)), lo, hi);
    return f2_pack(ex2_approx(lo), ex2_approx(hi));
}

// states beyond the last stay zero whatever the streams hold
__device__ __forceinline__ void keep_states(f2 (&h)[2], int first, int S) {
    float v[4];
    f2_unpack(h[0], v[0], v[1]);
    f2_unpack(h[1], v[2], v[3]);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = first + i < S ? v[i] : 0.f;
    h[0] = f2_pack(v[0], v[1]);
    h[1] = f2_pack(v[2], v[3]);
}

// entries of 16 bytes per lane group between a step's row and the next, so that the eight lanes that store at once meet no bank twice
template <int LPC> constexpr int kScanGroups = 32 / LPC + (LPC == 1 ? 0 : LPC == 2 ? 4 : LPC == 4 ? 2 : 1);

// One row's values of two channels as they are in memory, one word where they are neighbours that move as one (PAIRS).  They are taken
// apart and converted where they are used: an instruction next to the load would wait for it.
template <typename T, bool PAIRS> struct Two;
template <typename T> struct Two<T, false> {
    T v[2];
    __device__ __forceinline__ void load(const T* row, const int (&d)[2]) { v[0] = row[d[0]]; v[1] = row[d[1]]; }
    __device__ __forceinline__ float get(int c) const { return to_f32(v[c]); }
};
template <> struct Two<float, true> {
    float2 v;
    __device__ __forceinline__ void load(const float* row, const int (&d)[2]) { v = *reinterpret_cast<const float2*>(row + d[0]); }
    __device__ __forceinline__ float get(int c) const { return c ? v.y : v.x; }
};
template <> struct Two<__nv_bfloat16, true> {
    unsigned v;
    __device__ __forceinline__ void load(const __nv_bfloat16* row, const int (&d)[2]) { v = *reinterpret_cast<const unsigned*>(row + d[0]); }
    __device__ __forceinline__ float get(int c) const { return __uint_as_float(c ? v & 0xffff0000u : v << 16); }
};
template <bool PAIRS>
__device__ __forceinline__ void store_two(float* row, const int (&d)[2], const bool (&on)[2], const float (&v)[2]) {
    if (PAIRS) {
        if (on[0]) *reinterpret_cast<float2*>(row + d[0]) = make_float2(v[0], v[1]);
    } else {
        if (on[0]) row[d[0]] = v[0];
        if (on[1]) row[d[1]] = v[1];
    }
}
template <bool PAIRS>
__device__ __forceinline__ void store_two(__nv_bfloat16* row, const int (&d)[2], const bool (&on)[2], const float (&v)[2]) {
    if (PAIRS) {
        if (on[0]) *reinterpret_cast<__nv_bfloat162*>(row + d[0]) = __floats2bfloat162_rn(v[0], v[1]);
    } else {
        if (on[0]) row[d[0]] = from_f32<__nv_bfloat16>(v[0]);
        if (on[1]) row[d[1]] = from_f32<__nv_bfloat16>(v[1]);
    }
}

// the state of channel d before step t (a multiple of 8)
__device__ __forceinline__ void scan_checkpoint(const ScanParams& p, int n, int t, int d, bool on, int j, const f2 (&h)[2]) {
    const int row = scan_row(p.S);
    if (!on || 4 * j >= row) return;
    float* at = p.checkpoints + (((long long)n * ((p.L + kScanKeep - 1) / kScanKeep) + t / kScanKeep) * p.D + d) * row + 4 * j;
    ulonglong2 v;
    v.x = h[0];
    v.y = h[1];
    *reinterpret_cast<ulonglong2*>(at) = v;
}

#endif
}  // namespace fwp
