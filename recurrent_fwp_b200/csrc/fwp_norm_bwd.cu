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
// CTAs that an SM is to hold: 24 warps of the short forms with two sums per element, 16 with five, fewer of the long rows'
constexpr int norm_bwd_resident(int TPR, int EPT, bool FULL) {
    return TPR == 32 ? 2 : EPT == 4 || (EPT == 8 && !FULL) ? 24 / norm_bwd_warps(TPR) : EPT == 8 || !FULL ? 16 / norm_bwd_warps(TPR) : 1;
}

// Rows ahead of the one at work: two where shared memory has room for all the CTAs that an SM is to hold.  fp32 rows of 2049 to 4096 with the
// residual sum alone have room for two CTAs with one row ahead or one CTA with two: 107 and 112 us for 32 Mi elements at 4096, 153 and 180 us at 2052.
template <typename T, typename TR, int TPR, int EPT, int V, bool FULL>
struct NormBwdRing {
    static constexpr int SLOTS = TPR == 32 ? 8 : 1, ROW = TPR * EPT;
    static constexpr int kGy = ROW * sizeof(T), kGate = 2 * kGy, kRes = (FULL ? 3 : 2) * kGy, kGr = kRes + ROW * sizeof(TR), kStage = kGr + ROW * sizeof(TR);
    static constexpr int kRed = SLOTS > 1 ? SLOTS * ROW * 4 : 0;
    // of an SM's 227 KB, less 1 KB that every CTA takes for itself
    static constexpr int kRoom = (227 * 1024) / norm_bwd_resident(TPR, EPT, FULL) - 1024 - 4 * 8 * (TPR / 32);
    static constexpr int DEPTH = V != 4 ? 0 : 2 * SLOTS * kStage + kRed <= kRoom ? 2 : 1;
    static_assert(V != 4 || SLOTS * DEPTH * kStage + kRed <= kRoom, "the CTAs that an SM is to hold do not fit");
    static constexpr size_t bytes = (size_t)SLOTS * DEPTH * kStage + kRed;
};

// FULL: with a norm behind the block, a gate or a scale vector; without, only r = residual + number x
template <typename T, typename TR, int TPR, int EPT, int V, bool FULL>
__global__ void __launch_bounds__(norm_bwd_warps(TPR) * 32, norm_bwd_resident(TPR, EPT, FULL)) norm_bwd_kernel(NormParams p) {
    constexpr int SLOTS = TPR == 32 ? 8 : 1, NV = FULL ? 5 : 2, W = TPR / 32, P = EPT / 2;
    __shared__ float buf[TPR > 32 ? 8 * W : 1];
    using Ring = NormBwdRing<T, TR, TPR, EPT, V, FULL>;
    constexpr int DEPTH = Ring::DEPTH;
    extern __shared__ float4 norm_smem[];
    float (*red)[TPR * EPT] = reinterpret_cast<float (*)[TPR * EPT]>(norm_smem);
    unsigned char* ring = reinterpret_cast<unsigned char*>(norm_smem) + Ring::kRed + threadIdx.x / TPR * DEPTH * Ring::kStage;
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    f2 acc[NV][P];              // sums for weight, bias and, FULL, post_weight, post_bias, scale
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < P; i++) acc[k][i] = 0;
    const float inv = 1.f / p.D;
    int par = 0, at_stage = 0;
    const long long first = (long long)blockIdx.x * SLOTS + slot, by = (long long)gridDim.x * SLOTS;
    RowAt here(first, by, p.L), ahead = here;
    auto prefetch = [&](long long row, int stage) {
        if (row < p.rows) {
            auto at = [&](const Stream& s) { return ahead.of(s); };
            unsigned char* to = ring + stage * Ring::kStage;
            ring_issue<T, TPR, EPT>(to, static_cast<const T*>(p.x.p) + at(p.x), p.D, tid);
            if (p.gy.p) ring_issue<T, TPR, EPT>(to + Ring::kGy, static_cast<const T*>(p.gy.p) + at(p.gy), p.D, tid);
            if (FULL && p.gate.p) ring_issue<T, TPR, EPT>(to + Ring::kGate, static_cast<const T*>(p.gate.p) + at(p.gate), p.D, tid);
            if (p.res.p) ring_issue<TR, TPR, EPT>(to + Ring::kRes, static_cast<const TR*>(p.res.p) + at(p.res), p.D, tid);
            if (p.gr.p) ring_issue<TR, TPR, EPT>(to + Ring::kGr, static_cast<const TR*>(p.gr.p) + at(p.gr), p.D, tid);
        }
        cp_async_commit();
        ahead.next();
    };
    if constexpr (DEPTH > 0)
#pragma unroll
        for (int i = 0; i < DEPTH; i++) prefetch(first + i * by, i);
    float4 next_stats = first < p.rows ? *reinterpret_cast<const float4*>(p.stats + 4 * first) : make_float4(0.f, 0.f, 0.f, 0.f);
    for (long long row = first; row < p.rows; row += by, par ^= 1, here.next()) {
        auto at = [&](const Stream& s) { return here.of(s); };
        const float4 stats = next_stats;
        if (row + by < p.rows) next_stats = *reinterpret_cast<const float4*>(p.stats + 4 * (row + by));
        f2 x[P], r[P], g[P], gr[P];
        if constexpr (DEPTH > 0) cp_async_wait<DEPTH - 1>();
        const unsigned char* stage = ring + at_stage * Ring::kStage;
        auto load = [&](auto type, const Stream& s, int offset, auto& v) {
            using E = decltype(type);
            if constexpr (DEPTH > 0) row_load<TPR, EPT, V>(reinterpret_cast<const E*>(stage + offset), p.D, tid, v);
            else row_load<TPR, EPT, V>(static_cast<const E*>(s.p) + at(s), p.D, tid, v);
        };
        load(T(), p.x, 0, x);
#pragma unroll
        for (int i = 0; i < P; i++) r[i] = g[i] = gr[i] = 0;
        if (p.res.p) load(TR(), p.res, Ring::kRes, r);
        if (p.gy.p) load(T(), p.gy, Ring::kGy, g);
        if (p.gr.p) load(TR(), p.gr, Ring::kGr, gr);
        // t: what the gate multiplies, a: the gate's factor, da: its derivative, sc: the residual scale
        f2 t[FULL ? P : 1], a[FULL ? P : 1], da[FULL ? P : 1], sc[FULL ? P : 1], w[P];
        if constexpr (FULL) {
            if (p.pw) {
                const f2 s = f2_all(stats.y), m = f2_all(-stats.x);
                row_load<TPR, EPT, V>(p.pw, p.D, tid, w);
                if (p.pb) row_load<TPR, EPT, V>(p.pb, p.D, tid, t);
                else
#pragma unroll
                    for (int i = 0; i < P; i++) t[i] = 0;
#pragma unroll
                for (int i = 0; i < P; i++) {
                    x[i] = fmul2(fadd2(x[i], m), s);        // in the forward's order: rows may be large against their spread, or constant
                    t[i] = ffma2(x[i], w[i], t[i]);         // zero beyond the row, where w and b are
                }
            } else {
#pragma unroll
                for (int i = 0; i < P; i++) t[i] = x[i];
            }
            if (p.gate.p) {
                load(T(), p.gate, Ring::kGate, da);
                gate_factor_and_grad(p.act, da, a);
            } else {
#pragma unroll
                for (int i = 0; i < P; i++) a[i] = f2_all(1.f);
            }
            if (p.sv) row_load<TPR, EPT, V>(p.sv, p.D, tid, sc);
            else
#pragma unroll
                for (int i = 0; i < P; i++) sc[i] = f2_all(p.sval);
#pragma unroll
            for (int i = 0; i < P; i++) r[i] = ffma2(sc[i], fmul2(t[i], a[i]), r[i]);
        } else {
            const f2 s = f2_all(p.sval);
#pragma unroll
            for (int i = 0; i < P; i++) r[i] = ffma2(s, x[i], r[i]);
        }
        row_load<TPR, EPT, V>(p.w, p.D, tid, w);
        // here too the mean is taken off before the scaling
        const f2 rs = f2_all(stats.w), mean = f2_all(-stats.z);
        f2 s0 = 0, s1 = 0;
#pragma unroll
        for (int i = 0; i < P; i++) {
            r[i] = fmul2(fadd2(r[i], mean), rs);            // beyond the row g is zero
            acc[0][i] = ffma2(g[i], r[i], acc[0][i]);
            acc[1][i] = fadd2(acc[1][i], g[i]);
            g[i] = fmul2(g[i], w[i]);
            s0 = ffma2(g[i], r[i], s0);
            s1 = fadd2(s1, g[i]);
        }
        float s[2] = {f2_hsum(s0), f2_hsum(s1)};
        row_sum<TPR, 2>(s, buf + par * 4 * W);
        {
            const f2 m1 = f2_all(-s[0] * inv), m0 = f2_all(p.rms ? 0.f : -s[1] * inv);
#pragma unroll
            for (int i = 0; i < P; i++) g[i] = ffma2(rs, fadd2(ffma2(r[i], m1, g[i]), m0), gr[i]);
        }
        row_cut<TPR, EPT, V>(p.D, tid, g);
        if constexpr (DEPTH > 0) {              // every value of the stage has been used
            prefetch(row + DEPTH * by, at_stage);
            at_stage = at_stage + 1 == DEPTH ? 0 : at_stage + 1;
        }
        if (p.gres.p) row_store<TPR, EPT, V>(static_cast<TR*>(p.gres.p) + at(p.gres), p.D, tid, g);
        if constexpr (FULL) {
#pragma unroll
            for (int i = 0; i < P; i++) {
                acc[4][i] = ffma2(g[i], fmul2(t[i], a[i]), acc[4][i]);
                g[i] = fmul2(g[i], sc[i]);
            }
            if (p.gate.p) {
#pragma unroll
                for (int i = 0; i < P; i++) {
                    da[i] = fmul2(fmul2(g[i], t[i]), da[i]);
                    g[i] = fmul2(g[i], a[i]);
                }
                row_store<TPR, EPT, V>(static_cast<T*>(p.ggate.p) + at(p.ggate), p.D, tid, da);
            }
            if (p.pw) {
                row_load<TPR, EPT, V>(p.pw, p.D, tid, w);
                s0 = s1 = 0;
#pragma unroll
                for (int i = 0; i < P; i++) {
                    acc[2][i] = ffma2(g[i], x[i], acc[2][i]);
                    acc[3][i] = fadd2(acc[3][i], g[i]);
                    g[i] = fmul2(g[i], w[i]);
                    s0 = ffma2(g[i], x[i], s0);
                    s1 = fadd2(s1, g[i]);
                }
                s[0] = f2_hsum(s0);
                s[1] = f2_hsum(s1);
                row_sum<TPR, 2>(s, buf + par * 4 * W + 2 * W);
                const f2 q1 = f2_all(-s[0] * inv), q0 = f2_all(p.rms ? 0.f : -s[1] * inv), ps = f2_all(stats.y);
#pragma unroll
                for (int i = 0; i < P; i++) g[i] = fmul2(ps, fadd2(ffma2(x[i], q1, g[i]), q0));
            }
        } else {
            const f2 sv = f2_all(p.sval);
#pragma unroll
            for (int i = 0; i < P; i++) g[i] = fmul2(g[i], sv);
        }
        row_store<TPR, EPT, V>(static_cast<T*>(p.gx.p) + at(p.gx), p.D, tid, g);
    }
    float* part = p.part + (long long)blockIdx.x * p.D * NV;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        if constexpr (SLOTS == 1) {
            row_store<TPR, EPT, V>(part + (long long)k * p.D, p.D, tid, acc[k]);
        } else {
            __syncthreads();
            row_store<TPR, EPT, V>(red[slot], p.D, tid, acc[k]);
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

// threads and elements of each for a row of D; with five sums per element a warp has no registers for eight elements and a second CTA
struct NormBwdForm {
    int tpr, ept;
};
static NormBwdForm norm_bwd_form(int D, bool full) {
    if (D <= 256) return full ? NormBwdForm{64, 4} : NormBwdForm{32, 8};
    if (D <= 512) return {64, 8};
    if (D <= 1024) return {128, 8};
    if (D <= 2048) return {256, 8};
    return D <= 4096 ? NormBwdForm{256, 16} : NormBwdForm{512, 16};
}
// CTAs: those that stay resident, and no more partial sums than that
static int norm_bwd_ctas(long long rows, int D, bool full, long long sms) {
    const NormBwdForm f = norm_bwd_form(D, full);
    const long long resident = sms * norm_bwd_resident(f.tpr, f.ept, full), most = f.tpr == 32 ? ceil_div(rows, 8) : rows;
    return (int)(most < resident ? most : resident);
}

static int64_t norm_bwd_scratch(long long rows, int D, long long sms) {
    const int a = norm_bwd_ctas(rows, D, true, sms), b = norm_bwd_ctas(rows, D, false, sms);
    return (int64_t)(a > b ? a : b) * D * 5;
}

template <typename T, typename TR, int TPR, int EPT, bool FULL>
static int norm_bwd_launch(const NormParams& p, bool vec, int ctas, cudaStream_t st) {
    constexpr int threads = norm_bwd_warps(TPR) * 32;
    constexpr size_t b4 = NormBwdRing<T, TR, TPR, EPT, 4, FULL>::bytes, b1 = NormBwdRing<T, TR, TPR, EPT, 1, FULL>::bytes;
    if (vec) return launch_dependent_beside(norm_bwd_kernel<T, TR, TPR, EPT, 4, FULL>, p, dim3(ctas), threads, b4, st, "norm_bwd_kernel");
    return launch_dependent_beside(norm_bwd_kernel<T, TR, TPR, EPT, 1, FULL>, p, dim3(ctas), threads, b1, st, "norm_bwd_kernel");
}
template <typename T, typename TR, bool FULL>
static int norm_bwd_dispatch(const NormParams& p, bool vec, int ctas, cudaStream_t st) {
    switch (norm_bwd_form(p.D, FULL).tpr) {
        case 32: if constexpr (!FULL) return norm_bwd_launch<T, TR, 32, 8, FULL>(p, vec, ctas, st); break;
        case 64: if (p.D > 256) return norm_bwd_launch<T, TR, 64, 8, FULL>(p, vec, ctas, st);
                 if constexpr (FULL) return norm_bwd_launch<T, TR, 64, 4, FULL>(p, vec, ctas, st);
                 break;
        case 128: return norm_bwd_launch<T, TR, 128, 8, FULL>(p, vec, ctas, st);
        case 256: return p.D > 2048 ? norm_bwd_launch<T, TR, 256, 16, FULL>(p, vec, ctas, st) : norm_bwd_launch<T, TR, 256, 8, FULL>(p, vec, ctas, st);
        case 512: return norm_bwd_launch<T, TR, 512, 16, FULL>(p, vec, ctas, st);
    }
    return FWP_ERR_UNSUPPORTED;
}

}  // namespace fwp

using namespace fwp;

FWP_API int64_t fwp_block_norm_backward_scratch_floats(int N, int L, int D) {
    if (N <= 0 || L <= 0 || D <= 0 || D > kNormMaxD) return 0;
    return norm_bwd_scratch((long long)N * L, D, most_sms());
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
    const long long sms = sm_count() > 0 ? sm_count() : 148;
    if (!scratch || !aligned16(scratch) || scratch_floats < norm_bwd_scratch((long long)N * L, D, sms)) return FWP_ERR_SCRATCH;
    NormParams p = norm_params(N, L, D, x, residual, gate, scale_vector, scale_value, post_weight, post_bias, weight, bias, rms, gate_act);
    p.gy = stream_of(grad_y); p.gr = stream_of(grad_r); p.gx = stream_of(grad_x); p.gres = stream_of(grad_residual);
    p.ggate = stream_of(grad_gate);
    p.stats = const_cast<float*>(stats);
    p.part = scratch;
    bool vec = norm_vectors(p);
    for (const Stream* s : {&p.x, &p.gate, &p.gy, &p.gx, &p.ggate}) vec = vec && rows_aligned(*s, esz, 4 * esz);
    for (const Stream* s : {&p.res, &p.gr, &p.gres}) vec = vec && rows_aligned(*s, rsz, 4 * rsz);
    const bool full = p.pw || p.gate.p || p.sv;
    const int ctas = norm_bwd_ctas(p.rows, D, full, sms);
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
