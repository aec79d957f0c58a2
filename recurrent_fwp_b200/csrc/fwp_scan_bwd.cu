// Selective scan (sm_100a), backward.  With gy = gout silu(z):
//
//   g_t[s] = C_t[s] gy_t + exp(delta_{t+1} A[s]) g_{t+1}[s],  e_t = g_t exp(delta_t A) h_{t-1}
//   gB_t[s] = sum_ch g delta x,  gC_t[s] = sum_ch gy h,  p = sum_s g B,  q = sum_s e A
//   gx = delta p + skip gy,  gdelta = x p + q,  gA = sum_t e delta,  gz = gout y silu'(z)
//
// Tiles of eight steps, from the last to the first.  The state before a tile comes from the forward's checkpoints; the tile's decays and
// states are formed once and stay in registers (32 + 32 per lane).  A lane holds four states of one channel; sums over states end in the
// lane that loads and stores the (step, channel), as in the forward.  The sums over channels, gB and gC, halve their way through the lanes
// of a warp, meet the CTA's other warps in shared memory and leave as one row per CTA and step, added up in a fixed order by
// scan_bc_kernel: no atomics.
#include "fwp_scan.cuh"

namespace fwp {

constexpr float kLn2 = 0.6931471805599453f;
template <int LPC> constexpr int kBwdWarps = LPC == 16 ? 4 : 8;     // by shared memory: 2 x 4 LPC partial sums per warp and step

template <int LPC>
struct ScanBwdTile {
    static constexpr int W = kBwdWarps<LPC>, CW = 32 / LPC, S4 = 4 * LPC;
    float4 st[W][kScanKeep][CW];                // delta, x, gy
    float B[2][kScanKeep][S4];
    float C[2][kScanKeep][S4];
    float bc[2][W][kScanKeep][2 * S4];
};

// PASS = SCAN_ENDS: only exp(A delta) g of the span's first step, with nothing behind the span, and the sum of delta.
template <typename T, int LPC, bool RAGGED, int PASS>
__global__ void __launch_bounds__(kBwdWarps<LPC> * 32) scan_bwd_kernel(ScanParams p) {
    using Tile = ScanBwdTile<LPC>;
    constexpr int W = Tile::W, CW = Tile::CW, S4 = Tile::S4, TT = kScanKeep;
    constexpr int OS = LPC <= TT ? TT / LPC : 1;
    constexpr bool WHOLE = PASS == SCAN_WHOLE;
    __shared__ __align__(16) Tile sm;
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int grp = lane / LPC, j = lane % LPC;
    const int n = blockIdx.z, span = WHOLE ? blockIdx.y : blockIdx.y + 1;       // nothing in front of the first span asks for its end
    const int per = p.D / p.G, blocks = (per + CW * W - 1) / (CW * W);
    const int g = blockIdx.x / blocks;
    const int ch = ((blockIdx.x % blocks) * W + warp) * CW + grp;       // inside the group
    const bool on = ch < per, full = ch - grp + CW <= per;              // full: every lane of the warp has a channel
    const int d = g * per + (on ? ch : 0);
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
    const int t0 = span * p.span, tend = min(t0 + p.span, p.L), t1 = min(tend, len);
    const int first = LPC <= TT ? j * OS : j / 2;                        // the steps of a tile that this lane loads and stores
    const bool mine = on && (LPC <= TT || !(j & 1));
    const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
    const bool gated = p.z.p != nullptr;
    const T* x = static_cast<const T*>(p.x.p) + n * p.x.sN + d;
    const T* dt = static_cast<const T*>(p.dt.p) + n * p.dt.sN + d;
    const T* z = static_cast<const T*>(p.z.p) + n * p.z.sN + d;
    const T* gout = static_cast<const T*>(p.gout.p) + n * p.gout.sN + d;
    T* gx = static_cast<T*>(p.gx.p) + n * p.gx.sN + d;
    T* gdt = static_cast<T*>(p.gdt.p) + n * p.gdt.sN + d;
    T* gz = static_cast<T*>(p.gz.p) + n * p.gz.sN + d;
    const int row = scan_row(p.S);
    const float* keep = p.checkpoints + ((long long)n * ((p.L + TT - 1) / TT) * p.D + d) * row + 4 * j;
    const long long keep_step = (long long)p.D * row;
    const bool has = on && 4 * j < row;

    const long long spans_at = ((long long)n * p.spans + span) * p.D + d;
    f2 A[2], carry[2], dA[2] = {0, 0};
    {
        float a[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = on && 4 * j + i < p.S;
            a[i] = in ? p.A[(long long)d * p.S + 4 * j + i] * kLog2e : 0.f;
            s[i] = in && WHOLE && p.spans > 1 ? p.ends[spans_at * p.S + 4 * j + i] : 0.f;
        }
        A[0] = f2_pack(a[0], a[1]); A[1] = f2_pack(a[2], a[3]);
        carry[0] = f2_pack(s[0], s[1]); carry[1] = f2_pack(s[2], s[3]);
    }
    float gskip = 0.f, gbias = 0.f, dsum = 0.f;

    float rx[OS], rd[OS], rz[OS], rg[OS];
    float4 rh = {0.f, 0.f, 0.f, 0.f};
    constexpr int BC = (TT * S4 + W * 32 - 1) / (W * 32);
    float rB[BC], rC[BC];
    const T* Bp = static_cast<const T*>(p.B.p) + n * p.B.sN + g * p.B.sH;
    const T* Cp = static_cast<const T*>(p.C.p) + n * p.C.sN + g * p.C.sH;
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < OS; i++) {
            const int u = t + first + i;
            const bool in = mine && u < t1;
            rx[i] = WHOLE && in ? to_f32(x[u * p.x.sL]) : 0.f;
            rd[i] = in ? to_f32(dt[u * p.dt.sL]) : 0.f;
            rg[i] = in ? to_f32(gout[u * p.gout.sL]) : 0.f;
            rz[i] = in && gated ? to_f32(z[u * p.z.sL]) : 0.f;
        }
        if (WHOLE && has) rh = *reinterpret_cast<const float4*>(keep + (t / TT) * keep_step);
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int e = i * W * 32 + threadIdx.x, u = t + e / S4, s = e % S4;
            const bool in = e < TT * S4 && u < t1 && s < p.S;
            if (WHOLE) rB[i] = in ? to_f32(Bp[u * p.B.sL + s]) : 0.f;
            rC[i] = in ? to_f32(Cp[u * p.C.sL + s]) : 0.f;
        }
    };
    // the CTA's sums of the tile at t, from buffer `b`
    float* bc = p.bc + (((long long)blockIdx.x * p.N + n) * p.L) * (2 * S4);
    auto flush = [&](int t, int b) {
        for (int e = threadIdx.x; e < TT * 2 * S4; e += W * 32) {
            const int r = e / (2 * S4), c = e % (2 * S4);
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) a += sm.bc[b][w][r][c];
            if (t + r < t1) bc[(long long)(t + r) * (2 * S4) + c] = a;
        }
    };
    const int tiles = t1 > t0 ? (t1 - t0 + TT - 1) / TT : 0;
    if (tiles) fetch(t0 + (tiles - 1) * TT);
    int par = 0;
    for (int b = tiles - 1; b >= 0; b--, par ^= 1) {
        const int t = t0 + b * TT;
        float kx[OS], kr[OS], kd[OS], kz[OS], ks[OS], kg[OS], ky[OS];      // own pairs: x, dt + bias, delta, z, sigmoid(z), gout, gy
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int e = i * W * 32 + threadIdx.x;
            if (e < TT * S4) {
                if (WHOLE) sm.B[par][e / S4][e % S4] = rB[i];
                sm.C[par][e / S4][e % S4] = rC[i];
            }
        }
#pragma unroll
        for (int i = 0; i < OS; i++) {
            const int u = t + first + i;
            kx[i] = rx[i];
            kr[i] = rd[i] + bias;
            kd[i] = p.softplus ? softplus_(kr[i]) : kr[i];
            kd[i] = mine && u < t1 ? kd[i] : 0.f;
            kz[i] = rz[i];
            kg[i] = rg[i];
            ks[i] = gated ? sigmoidf_(kz[i]) : 1.f;
            ky[i] = gated ? kg[i] * silu_of(kz[i], ks[i]) : kg[i];
            if (LPC <= TT || !(j & 1)) sm.st[warp][first + i][grp] = make_float4(kd[i], kx[i], ky[i], 0.f);
            if (!WHOLE) dsum += kd[i];
        }
        f2 h[2] = {f2_pack(rh.x, rh.y), f2_pack(rh.z, rh.w)};
        const f2 h0[2] = {h[0], h[1]};
        __syncthreads();
        if (WHOLE && b < tiles - 1) flush(t + TT, par ^ 1);
        if (b > 0) fetch(t - TT);
        f2 a[TT][2], H[TT][2];
        float yv[TT];
#pragma unroll
        for (int r = 0; r < TT; r++) {
            const float4 s = sm.st[warp][r][grp];
            const f2 d2 = f2_pack(s.x, s.x);
            a[r][0] = exp2_pair(fmul2(d2, A[0]));
            a[r][1] = exp2_pair(fmul2(d2, A[1]));
            if (!WHOLE) continue;
            const float dx = s.x * s.y;
            const f2 x2 = f2_pack(dx, dx);
            const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B[par][r][4 * j]);
            const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][r][4 * j]);
            h[0] = ffma2(a[r][0], h[0], fmul2(x2, bb.x));
            h[1] = ffma2(a[r][1], h[1], fmul2(x2, bb.y));
            if (RAGGED) keep_states(h, 4 * j, p.S);
            H[r][0] = h[0];
            H[r][1] = h[1];
            if (gated) yv[r] = f2_hsum(ffma2(cc.y, h[1], fmul2(cc.x, h[0])));
        }
        if (WHOLE && gated) {
            sum_lanes<TT, LPC, 1>(yv, lane);
#pragma unroll
            for (int i = 0; i < OS; i++) {
                const int u = t + first + i;
                const float v = kg[i] * fmaf(skip, kx[i], yv[i]) * silu_grad_of(kz[i], ks[i]);
                if (mine && u < t1) gz[u * p.gz.sL] = from_f32<T>(v);
            }
        }
        float pv[TT], qv[TT];
#pragma unroll
        for (int r = TT - 1; r >= 0; r--) {
            const float4 s = sm.st[warp][r][grp];
            const f2 gy2 = f2_pack(s.z, s.z);
            const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][r][4 * j]);
            f2 gg[2] = {ffma2(cc.x, gy2, carry[0]), ffma2(cc.y, gy2, carry[1])};
            if (RAGGED) keep_states(gg, 4 * j, p.S);
            carry[0] = fmul2(a[r][0], gg[0]);
            carry[1] = fmul2(a[r][1], gg[1]);
            if (RAGGED) keep_states(carry, 4 * j, p.S);
            if (!WHOLE) continue;
            const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B[par][r][4 * j]);
            const float dx = s.x * s.y;
            const f2 x2 = f2_pack(dx, dx), d2 = f2_pack(s.x, s.x);
            const f2 e0 = fmul2(carry[0], r ? H[r ? r - 1 : 0][0] : h0[0]), e1 = fmul2(carry[1], r ? H[r ? r - 1 : 0][1] : h0[1]);
            pv[r] = f2_hsum(ffma2(gg[1], bb.y, fmul2(gg[0], bb.x)));
            qv[r] = f2_hsum(ffma2(e1, A[1], fmul2(e0, A[0])));
            dA[0] = ffma2(e0, d2, dA[0]);
            dA[1] = ffma2(e1, d2, dA[1]);
            float v[8];
            f2_unpack(fmul2(gg[0], x2), v[0], v[1]);
            f2_unpack(fmul2(gg[1], x2), v[2], v[3]);
            f2_unpack(fmul2(gy2, H[r][0]), v[4], v[5]);
            f2_unpack(fmul2(gy2, H[r][1]), v[6], v[7]);
            if (!full)
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = on ? v[i] : 0.f;
            sum_lanes<8, CW, LPC>(v, lane);
            if constexpr (CW <= 8) {
                constexpr int NV = 8 / CW;
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int k = grp * NV + i;
                    sm.bc[par][warp][r][(k >> 2) * S4 + 4 * j + (k & 3)] = v[i];
                }
            } else {
                constexpr int SH = CW / 8;
                const int k = grp / SH;
                if (grp % SH == 0) sm.bc[par][warp][r][(k >> 2) * S4 + 4 * j + (k & 3)] = v[0];
            }
        }
        if (WHOLE) {
            sum_lanes<TT, LPC, 1>(pv, lane);
            sum_lanes<TT, LPC, 1>(qv, lane);
#pragma unroll
            for (int i = 0; i < OS; i++) {
                const int u = t + first + i;
                float gd = fmaf(kx[i], pv[i], qv[i] * kLn2);
                if (p.softplus) gd *= sigmoidf_(kr[i]);
                if (mine && u < t1) {
                    gx[u * p.gx.sL] = from_f32<T>(fmaf(kd[i], pv[i], skip * ky[i]));
                    gdt[u * p.gdt.sL] = from_f32<T>(gd);
                    gskip = fmaf(ky[i], kx[i], gskip);
                    gbias += gd;
                }
            }
        }
        __syncwarp();           // the warp's st is read
    }
    if (WHOLE) {
        __syncthreads();
        if (tiles) flush(t0, par ^ 1);
        for (int u = max(t0, t1) + (LPC <= TT ? j : j / 2); mine && u < tend; u += LPC <= TT ? LPC : TT) {
            gx[u * p.gx.sL] = from_f32<T>(0.f);
            gdt[u * p.gdt.sL] = from_f32<T>(0.f);
            if (gated) gz[u * p.gz.sL] = from_f32<T>(0.f);
        }
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) {
            gskip += __shfl_xor_sync(0xffffffffu, gskip, o);
            gbias += __shfl_xor_sync(0xffffffffu, gbias, o);
        }
        float* sums = p.sums + ((long long)n * p.spans + span) * p.D * (p.S + 2);
        float v[4];
        f2_unpack(dA[0], v[0], v[1]);
        f2_unpack(dA[1], v[2], v[3]);
        if (!on) return;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * j + i < p.S) sums[(long long)d * p.S + 4 * j + i] = v[i];
        if (j == 0) {
            sums[(long long)p.D * p.S + d] = gskip;
            sums[(long long)p.D * (p.S + 1) + d] = gbias;
        }
    } else {
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) dsum += __shfl_xor_sync(0xffffffffu, dsum, o);
        if (!on) return;
        float v[4];
        f2_unpack(carry[0], v[0], v[1]);
        f2_unpack(carry[1], v[2], v[3]);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * j + i < p.S) p.ends[spans_at * p.S + 4 * j + i] = v[i];
        if (j == 0) p.dsums[spans_at] = dsum;
    }
}

// gB and gC from the CTAs' rows: one thread per (n, t, group, which, s), the CTAs of a group in order
struct ScanBcParams {
    ScanParams p;
    int S4, blocks;
};
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(ScanBcParams q) {
    const ScanParams& p = q.p;
    const int S4 = q.S4, blocks = q.blocks;
    griddep_wait();
    griddep_launch_dependents();
    const long long total = (long long)p.N * p.L * p.G * 2 * S4, step = (long long)p.N * p.L * 2 * S4;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int c = (int)(e % (2 * S4));
        const long long r = e / (2 * S4), nt = r / p.G;
        const int g = (int)(r - nt * p.G), n = (int)(nt / p.L), t = (int)(nt - (long long)n * p.L);
        const int which = c >= S4, s = c - which * S4;
        if (s >= p.S) continue;
        const bool in = !p.lengths || t < p.lengths[n];
        const float* at = p.bc + (long long)g * blocks * step + nt * (2 * S4) + c;
        float a = 0.f;
        if (in)
            for (int b = 0; b < blocks; b++) a += at[b * step];
        const Row4& o = which ? p.gCr : p.gBr;
        static_cast<T*>(o.p)[n * o.sN + g * o.sH + t * o.sL + s] = from_f32<T>(a);
    }
}

struct ScanBwdPlan {
    int span, spans, blocks;       // blocks: CTAs per group
};
static ScanBwdPlan scan_bwd_plan(int N, int L, int D, int S, int G) {
    const int lpc = scan_lanes(S), w = lpc == 16 ? 4 : 8, cw = 32 / lpc, per = D / G;
    const long long sms = sm_count() > 0 ? sm_count() : 148;
    ScanBwdPlan q;
    q.blocks = (int)ceil_div(per, cw * w);
    const long long ctas = (long long)N * G * q.blocks;
    const int forced = tune_get(T_SCAN_CHUNK, 0);
    int spans = 1;
    if (forced > 0) spans = (int)ceil_div(L, ceil_div(forced, kScanKeep) * kScanKeep);
    else if (ctas * 2 <= sms) spans = (int)(sms / ctas);
    const int most = (int)ceil_div(L, 8 * kScanKeep);
    if (!forced && spans > most) spans = most;
    if (spans > 4096) spans = 4096;
    q.span = (int)(ceil_div(ceil_div(L, spans), kScanKeep) * kScanKeep);
    q.spans = (int)ceil_div(L, q.span);
    return q;
}
static int64_t scan_bwd_scratch(const ScanBwdPlan& q, int N, int L, int D, int S, int G) {
    const int64_t S4 = 4 * scan_lanes(S);
    return (int64_t)G * q.blocks * N * L * 2 * S4 + (int64_t)N * q.spans * D * (S + 2) + (q.spans > 1 ? (int64_t)N * q.spans * D * (S + 1) : 0);
}

template <typename T, int LPC, bool RAGGED>
static int scan_bwd_launch(const ScanParams& p, const ScanBwdPlan& q, cudaStream_t st) {
    const unsigned gx = (unsigned)(p.G * q.blocks);
    constexpr int threads = kBwdWarps<LPC> * 32;
    if (q.spans > 1) {
        if (int rc = launch_dependent(scan_bwd_kernel<T, LPC, RAGGED, SCAN_ENDS>, p, dim3(gx, q.spans - 1, p.N), threads, 0, st, nullptr)) return rc;
        if (int rc = launch_scan_join(p, true, st)) return rc;
    }
    return launch_dependent(scan_bwd_kernel<T, LPC, RAGGED, SCAN_WHOLE>, p, dim3(gx, q.spans, p.N), threads, 0, st, "scan_bwd_kernel");
}
template <typename T>
static int scan_bwd_dispatch(const ScanParams& p, const ScanBwdPlan& q, cudaStream_t st) {
    const int lpc = scan_lanes(p.S);
    const bool ragged = p.S != 4 * lpc;
#define FWP_SCAN_BWD(LPC) (ragged ? scan_bwd_launch<T, LPC, true>(p, q, st) : scan_bwd_launch<T, LPC, false>(p, q, st))
    int rc;
    switch (lpc) {
        case 1: rc = FWP_SCAN_BWD(1); break;
        case 2: rc = FWP_SCAN_BWD(2); break;
        case 4: rc = FWP_SCAN_BWD(4); break;
        case 8: rc = FWP_SCAN_BWD(8); break;
        default: rc = FWP_SCAN_BWD(16);
    }
#undef FWP_SCAN_BWD
    if (rc) return rc;
    const long long values = (long long)p.N * p.L * p.G * 8 * lpc;
    const long long ctas = ceil_div(values, 256);
    ScanBcParams b = {p, 4 * lpc, q.blocks};
    return launch_dependent(scan_bc_kernel<T>, b, dim3((unsigned)(ctas < 65536 ? ctas : 65536)), 256, 0, st, nullptr);
}

}  // namespace fwp

using namespace fwp;

FWP_API int64_t fwp_selective_scan_backward_scratch_floats(int N, int L, int D, int S, int G, int device) {
    if (N <= 0 || L <= 0 || D <= 0 || S <= 0 || S > kScanMaxS || G <= 0 || D % G) return 0;
    DeviceGuard guard(device);
    return scan_bwd_scratch(scan_bwd_plan(N, L, D, S, G), N, L, D, S, G);
}

FWP_API int fwp_selective_scan_backward(int N, int L, int D, int S, int G, const fwp_tensor* x, const fwp_tensor* dt, const float* A,
                                        const fwp_tensor* B, const fwp_tensor* C, const float* skip, const fwp_tensor* z,
                                        const float* dt_bias, const int* lengths, const float* checkpoints, const fwp_tensor* grad_out,
                                        const fwp_tensor* grad_x, const fwp_tensor* grad_dt, float* grad_A, const fwp_tensor* grad_B,
                                        const fwp_tensor* grad_C, float* grad_skip, const fwp_tensor* grad_z, float* grad_dt_bias,
                                        float* scratch, int64_t scratch_floats, int softplus, int io_dtype, void* stream, int device) {
    const int esz = io_dtype == FWP_F32 ? 4 : 2;
    int rc;
    if ((rc = scan_check(N, L, D, S, G, x, dt, A, B, C, skip, z, dt_bias, lengths, io_dtype))) return rc;
    if (N && L && D) {
        for (const fwp_tensor* t : {grad_out, grad_x, grad_dt, grad_B, grad_C})
            if ((rc = check_tensor(t, esz, true))) return rc;
        if ((rc = check_tensor(grad_z, esz, given(z)))) return rc;
    }
    if (D && !grad_A) return FWP_ERR_NULL;
    if (!aligned4(grad_A) || !aligned4(grad_skip) || !aligned4(grad_dt_bias)) return FWP_ERR_ALIGN;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    cudaStream_t st = (cudaStream_t)stream;
    if (!N || !L || !D) {               // no steps: sums of nothing
        cudaError_t e = D ? cudaMemsetAsync(grad_A, 0, sizeof(float) * D * S, st) : cudaSuccess;
        if (e == cudaSuccess && D && grad_skip) e = cudaMemsetAsync(grad_skip, 0, sizeof(float) * D, st);
        if (e == cudaSuccess && D && grad_dt_bias) e = cudaMemsetAsync(grad_dt_bias, 0, sizeof(float) * D, st);
        return e == cudaSuccess ? FWP_OK : set_cuda_error(e);
    }
    if (!checkpoints) return FWP_ERR_NULL;
    if (!aligned16(checkpoints)) return FWP_ERR_ALIGN;
    const ScanBwdPlan q = scan_bwd_plan(N, L, D, S, G);
    if (!scratch || !aligned16(scratch) || scratch_floats < scan_bwd_scratch(q, N, L, D, S, G)) return FWP_ERR_SCRATCH;
    ScanParams p = scan_params(N, L, D, S, G, x, dt, A, B, C, skip, z, dt_bias, lengths, softplus);
    p.checkpoints = const_cast<float*>(checkpoints);
    p.gout = stream_of(grad_out); p.gx = stream_of(grad_x); p.gdt = stream_of(grad_dt); p.gz = stream_of(grad_z);
    p.gBr = row4(grad_B); p.gCr = row4(grad_C);
    p.span = q.span;
    p.spans = q.spans;
    p.bc = scratch;
    p.sums = p.bc + (int64_t)G * q.blocks * N * L * 8 * scan_lanes(S);
    p.ends = p.sums + (int64_t)N * q.spans * D * (S + 2);
    p.dsums = p.ends + (int64_t)N * q.spans * D * S;
    rc = io_dtype == FWP_F32 ? scan_bwd_dispatch<float>(p, q, st) : scan_bwd_dispatch<__nv_bfloat16>(p, q, st);
    if (rc) return rc;
    const long long ds = (long long)D * S;
    ColumnSums s = {p.sums, N * q.spans, ds + 2 * D, {grad_A, grad_skip, grad_dt_bias}, {ds, ds + D, ds + 2 * D}};
    return launch_column_sums(s, st);
}
