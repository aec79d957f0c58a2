// Selective scan (sm_100a), forward and single steps.
//
//   delta_t = softplus(dt_t + bias),  h_t[s] = exp(delta_t A[s]) h_{t-1}[s] + delta_t x_t B_t[s]
//   y_t = sum_s C_t[s] h_t[s] + skip x_t,  out_t = y_t z_t sigmoid(z_t)
//
// Every channel is a recurrence of its own over S states, B and C are shared by the channels of a group.  A lane holds four
// states of two channels, LPC lanes all of them (S <= 4 LPC).  With LPC steps in hand the sums over s cost LPC - 1 shuffles and leave each
// lane with the value of one step; that lane loads x, dt, z for it and stores its output, so y goes through no memory.
//
// The exponentials bound it: S per (step, channel), 16 a clock and SM.  At 8 x 2048 x 2048 (bf16, S = 16) that is 115 us, and 29 us more for
// softplus and silu; measured 293 us, 321 us with checkpoints.  With one channel per lane shared memory was the limit (B and C read for 8
// channels at a time, 89 % of the pipe, 383 us); with two it is the latency of 1.7 warps per scheduler (exponential unit 48 %, issue 48 %,
// shared memory 47 %; four CTAs of 128 registers would fit, there are 256 for 148 SMs).
#include "fwp_scan.cuh"

namespace fwp {

constexpr int kScanWarps = 4;

template <int LPC>
struct ScanTile {
    static constexpr int GR = 32 / LPC, CW = 2 * GR;        // lane groups and channels per warp
    static constexpr int OS = LPC == 1 ? 8 : LPC <= 4 ? 4 : 16 / LPC;   // steps per lane and tile, of two channels each
    static constexpr int TT = OS * LPC;                     // steps per tile
    static constexpr int S4 = 4 * LPC;
    float4 st[kScanWarps][TT][kScanGroups<LPC>];                          // delta and delta x of a lane group's two channels
    float B[2][TT][S4];
    float C[2][TT][S4];
};

// One span of time of one warp's channels.  PASS = SCAN_ENDS: only the state that the span leaves behind, starting from zero, and
// the sum of delta, for joining spans (scan_join_kernel).
template <typename T, int LPC, bool RAGGED, bool PAIRS, int PASS>
__global__ void __launch_bounds__(kScanWarps * 32, PASS == SCAN_WHOLE ? 4 : 3) scan_fwd_kernel(ScanParams p) {
    using Tile = ScanTile<LPC>;
    constexpr int CW = Tile::CW, OS = Tile::OS, TT = Tile::TT, S4 = Tile::S4, NT = kScanWarps * 32;
    constexpr bool WHOLE = PASS == SCAN_WHOLE;
    __shared__ __align__(16) Tile sm;
    griddep_wait();         // and no early launch of the next kernel: its CTAs would take this one's places unevenly (a prompt of 16384: 448 -> 621 us)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int grp = lane / LPC, j = lane % LPC;             // two channels; their states 4 j ... 4 j + 3, their steps j, j + LPC ...
    const int n = blockIdx.z, span = blockIdx.y;
    const int per = p.D / p.G, blocks = (per + CW * kScanWarps - 1) / (CW * kScanWarps);
    const int g = blockIdx.x / blocks;
    const int ch = ((blockIdx.x % blocks) * kScanWarps + warp) * CW + 2 * grp;     // inside the group
    const bool on[2] = {ch < per, ch + 1 < per};
    // a lane without a channel reads the last one's rows (the last pair's where they move as pairs: an even channel) and writes nothing
    const int first = min(ch, per - (PAIRS ? 2 : 1));
    const int d[2] = {g * per + first, g * per + min(first + 1, per - 1)};
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
    const int t0 = span * p.span, tend = min(t0 + p.span, p.L), t1 = min(tend, len);
    const bool gated = p.z.p != nullptr;
    const T* x = static_cast<const T*>(p.x.p) + n * p.x.sN;
    const T* dt = static_cast<const T*>(p.dt.p) + n * p.dt.sN;
    const T* z = static_cast<const T*>(p.z.p) + n * p.z.sN;
    T* out = static_cast<T*>(p.out.p) + n * p.out.sN;

    f2 A[2][2], h[2][2];
    float bias[2], skip[2], dsum[2] = {0.f, 0.f};
    const long long spans_at = ((long long)n * p.spans + span) * p.D;       // this span's rows in the workspace
#pragma unroll
    for (int c = 0; c < 2; c++) {
        bias[c] = p.dt_bias ? p.dt_bias[d[c]] : 0.f;
        skip[c] = p.skip ? p.skip[d[c]] : 0.f;
        float a[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int st = 4 * j + i;
            a[i] = st < p.S ? rate_of(p.A[(long long)d[c] * p.S + st]) : 0.f;
            s[i] = 0.f;
            if (WHOLE && st < p.S) {
                if (p.spans > 1) s[i] = p.ends[(spans_at + d[c]) * p.S + st];
                else if (p.state) s[i] = p.state[n * p.state_sN + d[c] * p.state_sD + st];
            }
        }
        A[c][0] = f2_pack(a[0], a[1]); A[c][1] = f2_pack(a[2], a[3]);
        h[c][0] = f2_pack(s[0], s[1]); h[c][1] = f2_pack(s[2], s[3]);
    }

    // The next tile's streams, as they are in memory: a conversion here would wait for the load.  Rows behind the end repeat the last one.
    Two<T, PAIRS> rx[OS], rd[OS], rz[OS];
    constexpr int BC = (TT * S4 + NT - 1) / NT;
    static_assert((TT * S4) % NT == 0 || TT * S4 < NT, "whole passes over a tile of B and C");
    T rB[BC], rC[BC];
    const int bc_row = threadIdx.x / S4, bc_s = threadIdx.x % S4;
    const bool bc_on = (!RAGGED || bc_s < p.S) && bc_row < TT;
    const T* Bp = static_cast<const T*>(p.B.p) + n * p.B.sN + g * p.B.sH + (bc_on ? bc_s : 0);
    const T* Cp = static_cast<const T*>(p.C.p) + n * p.C.sN + g * p.C.sH + (bc_on ? bc_s : 0);
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < OS; i++) {
            const int u = min(t + j + i * LPC, t1 - 1);
            rd[i].load(dt + u * p.dt.sL, d);
            rx[i].load(x + u * p.x.sL, d);
            if (WHOLE && gated) rz[i].load(z + u * p.z.sL, d);
        }
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int u = min(t + bc_row + i * (NT / S4), t1 - 1);
            rB[i] = Bp[u * p.B.sL];
            if (WHOLE) rC[i] = Cp[u * p.C.sL];
        }
    };
    if (t0 < t1) fetch(t0);
    int par = 0;
    for (int t = t0; t < t1; t += TT, par ^= 1) {
        Two<T, PAIRS> kx[OS], kz[OS];
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int r = bc_row + i * (NT / S4);
            if (TT * S4 >= NT || bc_row < TT) {
                const bool in = bc_on && t + r < t1;
                sm.B[par][r][bc_s] = in ? to_f32(rB[i]) : 0.f;
                if (WHOLE) sm.C[par][r][bc_s] = in ? to_f32(rC[i]) : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < OS; i++) {
            const bool in = t + j + i * LPC < t1;           // a step behind the end leaves the state as it is
            float dl[2], dx[2];
            kx[i] = rx[i];
            if (WHOLE && gated) kz[i] = rz[i];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                dl[c] = rd[i].get(c) + bias[c];
                if (p.softplus) dl[c] = softplus_(dl[c]);
                dl[c] = in ? dl[c] : 0.f;
                dx[c] = in ? dl[c] * rx[i].get(c) : 0.f;
                if (!WHOLE) dsum[c] += dl[c];
            }
            sm.st[warp][j + i * LPC][grp] = make_float4(dl[0], dx[0], dl[1], dx[1]);
        }
        __syncthreads();            // B and C of this tile are there; those of the tile before last are free
        if (t + TT < t1) fetch(t + TT);
#pragma unroll
        for (int i = 0; i < OS; i++) {
            float v[2][LPC];
#pragma unroll
            for (int k = 0; k < LPC; k++) {
                const int r = i * LPC + k;
                if (WHOLE && r % kScanKeep == 0 && p.checkpoints && t + r < t1) {
                    scan_checkpoint(p, n, t + r, d[0], on[0], j, h[0]);
                    scan_checkpoint(p, n, t + r, d[1], on[1], j, h[1]);
                }
                const float4 s = sm.st[warp][r][grp];
                const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&sm.B[par][r][4 * j]);
                ulonglong2 cc = {};
                if (WHOLE) cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][r][4 * j]);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float dl = c ? s.z : s.x, dx = c ? s.w : s.y;
                    const f2 d2 = f2_pack(dl, dl), x2 = f2_pack(dx, dx);
                    const f2 e0 = decay_pair(d2, A[c][0]), e1 = decay_pair(d2, A[c][1]);
                    h[c][0] = ffma2(e0, h[c][0], fmul2(x2, b.x));
                    h[c][1] = ffma2(e1, h[c][1], fmul2(x2, b.y));
                    if (RAGGED) keep_states(h[c], 4 * j, p.S);
                    if (WHOLE) v[c][k] = f2_hsum(ffma2(cc.y, h[c][1], fmul2(cc.x, h[c][0])));
                }
            }
            if (WHOLE) {
                const int u = t + j + i * LPC;
                float y[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    sum_lanes<LPC, LPC, 1>(v[c], lane);
                    y[c] = fmaf(skip[c], kx[i].get(c), v[c][0]);
                    const float zz = gated ? kz[i].get(c) : 0.f;
                    if (gated) y[c] *= silu_of(zz, sigmoidf_(zz));
                }
                if (u < t1) store_two<PAIRS>(out + u * p.out.sL, d, on, y);
            }
        }
        __syncwarp();               // the warp's st is read
    }
    if (WHOLE) {
        const float zero[2] = {0.f, 0.f};
        for (int u = max(t0, t1) + j; u < tend; u += LPC) store_two<PAIRS>(out + u * p.out.sL, d, on, zero);
    }
    // what the span leaves
#pragma unroll
    for (int c = 0; c < 2; c++) {
        if (on[c] && (!WHOLE || (span == p.spans - 1 && p.state))) {
            float s[4];
            f2_unpack(h[c][0], s[0], s[1]); f2_unpack(h[c][1], s[2], s[3]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int st = 4 * j + i;
                if (st >= p.S) continue;
                if (!WHOLE) p.ends[(spans_at + d[c]) * p.S + st] = s[i];
                else p.state[n * p.state_sN + d[c] * p.state_sD + st] = s[i];
            }
        }
        if (!WHOLE) {
            // the lanes of a channel hold sums over different steps
#pragma unroll
            for (int o = 1; o < LPC; o <<= 1) dsum[c] += __shfl_xor_sync(0xffffffffu, dsum[c], o);
            if (on[c] && j == 0) p.dsums[spans_at + d[c]] = dsum[c];
        }
    }
}

// Joins the spans of a sequence: h_{k+1} = exp(A sum delta_k) h_k + end_k, forwards from the state, backwards (the gradient's recurrence) from
// zero.  The start of each span replaces its end in the workspace; the last one's end is not needed.  One thread per state, spans in
// order, eight of them loaded ahead.
struct ScanJoinParams {
    ScanParams p;
    int backwards;
};
// exp(A sum delta) h from the root of the factor.  Where states grow the factor of a span may pass the range of a float though no step's does and
// its product with h does not either, so it is taken in two halves; a zero stays zero and an infinity stays one, as step after step leaves them.
__device__ __forceinline__ float over_span(float h, float root) { return h == 0.f || isinf(h) ? h : h * root * root; }
__global__ void __launch_bounds__(256) scan_join_kernel(ScanJoinParams q) {
    const ScanParams& p = q.p;
    griddep_wait();
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x, per_seq = (long long)p.D * p.S;
    if (e >= per_seq) return;
    const int n = blockIdx.y, d = (int)(e / p.S), s = (int)(e - (long long)d * p.S);
    const float a = rate_of(p.A[e]);
    float h = !q.backwards && p.state ? p.state[n * p.state_sN + d * p.state_sD + s] : 0.f;
    float* ends = p.ends + (long long)n * p.spans * per_seq + e;
    const float* dsum = p.dsums + (long long)n * p.spans * p.D + d;
    const int from = q.backwards ? p.spans - 1 : 0, by = q.backwards ? -1 : 1;
    for (int k0 = 0; k0 < p.spans; k0 += 8) {
        float end[8], f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool on = k0 + i < p.spans - 1;
            const long long k = from + by * (k0 + i);
            end[i] = on ? ends[k * per_seq] : 0.f;
            f[i] = on ? decay_of(0.5f * dsum[k * p.D], a) : 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (k0 + i < p.spans) ends[(from + by * (k0 + i)) * per_seq] = h;
            h = over_span(h, f[i]) + end[i];
        }
    }
}
int launch_scan_join(const ScanParams& p, bool backwards, cudaStream_t st) {
    const ScanJoinParams q = {p, backwards ? 1 : 0};
    return launch_dependent(scan_join_kernel, q, dim3((unsigned)ceil_div((long long)p.D * p.S, 256), p.N), 256, 0, st, nullptr);
}

// One step: the state is read and written once, and that is the work: 16.8 MB for 64 sequences of 2048 channels and 16 states, 6.5 us with
// two sequences to a thread, which halves the reads of A (7.8 with one, 7.0 with four at twice the registers).  Everything is loaded before
// anything is converted or stored.  VEC: rows of the state, of B and of C move in pieces of four.
constexpr int kStepSeqs = 2;
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(128) scan_step_kernel(ScanParams p) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, j = lane % LPC;
    const int ch = (int)(((long long)blockIdx.x * 128 + threadIdx.x) / LPC);
    const bool on = ch < p.D;
    const int d = on ? ch : 0, g = d / (p.D / p.G);
    const int j4 = 4 * j < p.S ? 4 * j : 0;         // a lane without states reads the first four and writes nothing
    T x[kStepSeqs], dt[kStepSeqs], z[kStepSeqs];
    RawVec<T, VEC ? 4 : 1> B[kStepSeqs][VEC ? 1 : 4], C[kStepSeqs][VEC ? 1 : 4];
    float h[kStepSeqs][4];
    bool live[kStepSeqs];
#pragma unroll
    for (int q = 0; q < kStepSeqs; q++) {
        const int at = blockIdx.y * kStepSeqs + q, n = min(at, p.N - 1);
        live[q] = at < p.N && (!p.lengths || p.lengths[n] > 0);
        x[q] = static_cast<const T*>(p.x.p)[n * p.x.sN + d];
        dt[q] = static_cast<const T*>(p.dt.p)[n * p.dt.sN + d];
        if (p.z.p) z[q] = static_cast<const T*>(p.z.p)[n * p.z.sN + d];
        const T* b = static_cast<const T*>(p.B.p) + n * p.B.sN + g * p.B.sH + j4;
        const T* c = static_cast<const T*>(p.C.p) + n * p.C.sN + g * p.C.sH + j4;
#pragma unroll
        for (int i = 0; i < (VEC ? 1 : 4); i++) {
            const int s = min(i, p.S - 1 - j4);
            B[q][i].load(b + s);
            C[q][i].load(c + s);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) h[q][i] = 0.f;
        if (p.state) {
            const float* st = p.state + n * p.state_sN + d * p.state_sD + j4;
            if (VEC) load_vec<4>(st, h[q]);
            else
#pragma unroll
                for (int i = 0; i < 4; i++) h[q][i] = st[min(i, p.S - 1 - j4)];
        }
    }
    float a[4];
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] = 4 * j + i < p.S ? rate_of(p.A[(long long)d * p.S + 4 * j + i]) : 0.f;
    const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
    float y[kStepSeqs];
#pragma unroll
    for (int q = 0; q < kStepSeqs; q++) {
        const int n = blockIdx.y * kStepSeqs + q;
        float e = to_f32(dt[q]) + bias;
        if (p.softplus) e = softplus_(e);
        const float ex = e * to_f32(x[q]);
        y[q] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * j + i < p.S) {
                h[q][i] = fmaf(decay_of(e, a[i]), h[q][i], ex * (VEC ? B[q][0].get(i) : B[q][VEC ? 0 : i].get(0)));
                y[q] = fmaf(VEC ? C[q][0].get(i) : C[q][VEC ? 0 : i].get(0), h[q][i], y[q]);
            }
        if (!live[q] || !on || !p.state) continue;
        float* st = p.state + n * p.state_sN + d * p.state_sD + 4 * j;
        if (VEC) {
            if (4 * j < p.S) store_vec<4>(st, h[q]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * j + i < p.S) st[i] = h[q][i];
        }
    }
#pragma unroll
    for (int q = 0; q < kStepSeqs; q++) {
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) y[q] += __shfl_xor_sync(0xffffffffu, y[q], o);
        const int n = blockIdx.y * kStepSeqs + q;
        if (!on || j || n >= p.N) continue;
        float v = fmaf(skip, to_f32(x[q]), y[q]);
        if (p.z.p) v *= silu_of(to_f32(z[q]), sigmoidf_(to_f32(z[q])));
        static_cast<T*>(p.out.p)[n * p.out.sN + d] = from_f32<T>(live[q] ? v : 0.f);
    }
}

// ------------------------------------------------------------------------------------------------------------ host side
struct ScanPlan {
    int span, spans;        // steps per span, a multiple of every form's tile
};
static ScanPlan scan_plan(int N, int L, int D, int S, int G) {
    const int cta = 64 / scan_lanes(S) * kScanWarps, tile = 32;
    const long long sms = sm_count() > 0 ? sm_count() : 148, ctas = (long long)N * G * ceil_div(D / G, cta);
    const int forced = tune_get(T_SCAN_CHUNK, 0);
    long long spans = 1;
    // Spans side by side form the exponentials of a step twice, so they have to bring more than twice the CTAs, of which an SM holds four and is busy with two.
    if (forced > 0) spans = ceil_div(L, ceil_div(forced, tile) * tile);
    else if (ctas * 3 <= sms * 2) {
        spans = sms * 2 / ctas;
        const long long most = ceil_div(L, L <= 512 ? tile : 2 * tile);        // the join goes through them one by one: 1 x 4096 x 64, spans of 32 and 64: 53 and 37 us
        if (spans > most) spans = most;
    }
    if (spans > 2048) spans = 2048;         // rounded up to the tile they end within 2^16 of the sequence: see kMaxSteps
    auto cut = [&](long long n) {
        ScanPlan q;
        q.span = (int)(ceil_div(ceil_div(L, n), tile) * tile);
        q.spans = (int)ceil_div(L, q.span);
        return q;
    };
    const ScanPlan q = cut(spans);
    if (forced > 0 || q.spans == 1) return q;
    // And they have to shorten the chain: a span is walked twice, 1.23 times as long a step where SMs have two CTAs, and the two launches beside the
    // first take about 48 steps' time.  One launch against spans (bf16, 16 states, 2048 channels): one sequence of 96 steps 11.8 and 12.0 us, 112 steps
    // 13.4 and 12.6, 256 steps 27.8 and 16.1; two of 160 steps 18.1 and 19.7, 192 steps 21.4 and 19.9; three of 320 steps 34.4 and 37.7, 384 steps 40.8 and 38.4.
    const long long walked = 2LL * q.span, beside = ctas * q.spans > sms ? ctas * q.spans - sms : 0;
    return walked + walked * beside * 23 / (sms * 100) + 48 > L ? cut(1) : q;
}

template <typename T, int LPC, bool RAGGED, bool PAIRS>
static int scan_launch(const ScanParams& p, cudaStream_t st) {
    const unsigned gx = (unsigned)(p.G * ceil_div(p.D / p.G, 64 / LPC * kScanWarps));
    if (p.spans > 1) {
        if (int rc = launch_dependent(scan_fwd_kernel<T, LPC, RAGGED, PAIRS, SCAN_ENDS>, p, dim3(gx, p.spans - 1, p.N), kScanWarps * 32, 0, st, nullptr)) return rc;
        if (int rc = launch_scan_join(p, false, st)) return rc;
    }
    return launch_dependent(scan_fwd_kernel<T, LPC, RAGGED, PAIRS, SCAN_WHOLE>, p, dim3(gx, p.spans, p.N), kScanWarps * 32, 0, st, "scan_fwd_kernel");
}
template <typename T, int LPC>
static int scan_lanes_launch(const ScanParams& p, cudaStream_t st) {
    if (p.L == 1 && !p.checkpoints) {
        const dim3 grid((unsigned)ceil_div((long long)p.D * LPC, 128), (unsigned)ceil_div(p.N, kStepSeqs));
        if (p.state_vec) return launch_dependent(scan_step_kernel<T, LPC, true>, p, grid, 128, 0, st, "scan_step_kernel");
        return launch_dependent(scan_step_kernel<T, LPC, false>, p, grid, 128, 0, st, "scan_step_kernel");
    }
    if (p.S != 4 * LPC) return scan_launch<T, LPC, true, false>(p, st);
    return p.pairs ? scan_launch<T, LPC, false, true>(p, st) : scan_launch<T, LPC, false, false>(p, st);
}
template <typename T>
static int scan_dispatch(const ScanParams& p, cudaStream_t st) {
    switch (scan_lanes(p.S)) {
        case 1: return scan_lanes_launch<T, 1>(p, st);
        case 2: return scan_lanes_launch<T, 2>(p, st);
        case 4: return scan_lanes_launch<T, 4>(p, st);
        case 8: return scan_lanes_launch<T, 8>(p, st);
    }
    return scan_lanes_launch<T, 16>(p, st);
}

}  // namespace fwp

using namespace fwp;

FWP_API int64_t fwp_selective_scan_checkpoint_floats(int N, int L, int D, int S) {
    if (N <= 0 || L <= 0 || D <= 0 || S <= 0 || S > kScanMaxS) return 0;
    return (int64_t)N * ceil_div(L, kScanKeep) * D * scan_row(S);
}

static int64_t scan_scratch(const ScanPlan& q, int N, int D, int S) {
    return q.spans > 1 ? (int64_t)N * q.spans * D * (S + 1) : 0;
}

FWP_API int64_t fwp_selective_scan_scratch_floats(int N, int L, int D, int S, int G, int device) {
    if (N <= 0 || L <= 1 || D <= 0 || S <= 0 || S > kScanMaxS || G <= 0 || D % G) return 0;
    DeviceGuard guard(device);
    return scan_scratch(scan_plan(N, L, D, S, G), N, D, S);
}

FWP_API int fwp_selective_scan_forward(int N, int L, int D, int S, int G, const fwp_tensor* x, const fwp_tensor* dt, const float* A,
                                       const fwp_tensor* B, const fwp_tensor* C, const float* skip, const fwp_tensor* z,
                                       const float* dt_bias, const fwp_tensor* state, const int* lengths, const fwp_tensor* out,
                                       float* checkpoints, float* scratch, int64_t scratch_floats, int softplus, int io_dtype,
                                       void* stream, int device) {
    const int esz = io_dtype == FWP_F32 ? 4 : 2;
    int rc;
    if ((rc = scan_check(N, L, D, S, G, x, dt, A, B, C, skip, z, dt_bias, lengths, io_dtype)) || !N || !L || !D) return rc;
    if ((rc = check_tensor(state, 4, false)) || (rc = check_tensor(out, esz, true))) return rc;
    if (!aligned16(checkpoints)) return FWP_ERR_ALIGN;
    DeviceGuard guard(device);
    if (guard.status) return guard.status;
    ScanParams p = scan_params(N, L, D, S, G, x, dt, A, B, C, skip, z, dt_bias, lengths, softplus);
    p.out = stream_of(out);
    if (given(state)) {
        p.state = static_cast<float*>(state->data);
        p.state_sN = state->stride[0];
        p.state_sD = state->stride[2];
        // rows of the state, and of B and C, in pieces of four
        p.state_vec = S % 4 == 0 && aligned16(p.state) && p.state_sN % 4 == 0 && p.state_sD % 4 == 0;
        for (const Row4* r : {&p.B, &p.C})
            p.state_vec = p.state_vec && reinterpret_cast<uintptr_t>(r->p) % (4 * esz) == 0 && r->sN % 4 == 0 && r->sH % 4 == 0;
    }
    p.checkpoints = checkpoints;
    p.pairs = D / G % 2 == 0 && rows_aligned(p.x, esz, 2 * esz) && rows_aligned(p.dt, esz, 2 * esz) && rows_aligned(p.z, esz, 2 * esz) &&
              rows_aligned(p.out, esz, 2 * esz);
    const ScanPlan q = scan_plan(N, L, D, S, G);
    p.span = q.span;
    p.spans = q.spans;
    if (L > 1 || checkpoints) {
        const int64_t need = L > 1 ? scan_scratch(q, N, D, S) : 0;
        if (need && (!scratch || !aligned16(scratch) || scratch_floats < need)) return FWP_ERR_SCRATCH;
        p.ends = scratch;
        p.dsums = scratch + (int64_t)N * q.spans * D * S;
    }
    cudaStream_t st = (cudaStream_t)stream;
    return io_dtype == FWP_F32 ? scan_dispatch<float>(p, st) : scan_dispatch<__nv_bfloat16>(p, st);
}
