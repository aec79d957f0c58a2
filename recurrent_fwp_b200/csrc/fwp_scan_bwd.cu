// Selective scan (sm_100a), backward.  With gy = gout silu(z):
//
//   g_t[s] = C_t[s] gy_t + exp(delta_{t+1} A[s]) g_{t+1}[s],  e_t = g_t exp(delta_t A) h_{t-1}
//   gB_t[s] = sum_ch g delta x,  gC_t[s] = sum_ch gy h,  p = sum_s g B,  q = sum_s e A
//   gx = delta p + skip gy,  gdelta = x p + q,  gA = sum_t e delta,  gz = gout y silu'(z)
//
// Tiles of eight steps, from the last to the first.  The state before a tile comes from the forward's checkpoints.  A lane holds four states
// of two channels, as in the forward; of half a tile it keeps decays and states in registers (32 + 32), so the first half's are formed
// twice: twelve exponentials per state and tile where eight steps in registers would take eight, for two channels at a time, which
// halves the reads of B and C and the shuffles below.  Sums over states end in the lane that loads and stores the (step, channel).  The
// sums over channels, gB and gC, halve their way through the lanes of a warp, meet the CTA's other warps in shared memory and leave as one
// row per CTA and step, added up in a fixed order by scan_bc_kernel: no atomics.  8 x 2048 x 2048 (bf16, S = 16): 874 us, 216 instructions per
// 16 channels and step at 47 % issue with 1.7 warps per scheduler; 1985 us with one channel per lane and whole tiles in registers.
#include <type_traits>
#include "fwp_scan.cuh"

namespace fwp {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kBwdWarps = 4;
constexpr int kHalf = kScanKeep / 2;

template <int LPC>
struct ScanBwdTile {
    static constexpr int GR = 32 / LPC, S4 = 4 * LPC;
    float4 st[kBwdWarps][kScanKeep][kScanGroups<LPC>];      // delta and delta x of a lane group's two channels
    float2 gy[kBwdWarps][kScanKeep][GR + 4];
    float B[2][kScanKeep][S4];
    float C[2][kScanKeep][S4];
    float bc[2][kBwdWarps][kScanKeep][2 * S4];
    float4 dA[kBwdWarps][2][32];                            // sums of gA over more tiles than the registers take
};

// what a lane loads and stores of a half tile's 4 x 2 (step, channel) pairs: STEPS steps of NC channels
template <int LPC>
struct ScanOwn {
    static constexpr int NC = LPC <= 4 ? 2 : 1, STEPS = LPC <= 4 ? 4 / LPC : 1;
    static __device__ __forceinline__ int step(int j) { return LPC <= 4 ? j * STEPS : LPC == 8 ? j / 2 : j / 4; }
    static __device__ __forceinline__ int channel(int j) { return LPC <= 4 ? 0 : LPC == 8 ? j & 1 : (j >> 1) & 1; }
    static __device__ __forceinline__ bool first(int j) { return LPC <= 8 || !(j & 1); }      // two lanes share a pair at LPC = 16
};
template <typename T> struct One {
    T v;
    __device__ __forceinline__ void load(const T* row, const int (&d)[2]) { v = row[d[0]]; }
    __device__ __forceinline__ float get(int) const { return to_f32(v); }
};

// PASS = SCAN_ENDS: only exp(A delta) g of the span's first step, with nothing behind the span, and the sum of delta.
template <typename T, int LPC, bool RAGGED, bool PAIRS, int PASS>
__global__ void __launch_bounds__(kBwdWarps * 32, 2) scan_bwd_kernel(ScanParams p) {
    using Tile = ScanBwdTile<LPC>;
    using Own = ScanOwn<LPC>;
    using Raw = typename std::conditional<Own::NC == 2, Two<T, PAIRS>, One<T>>::type;
    constexpr int GR = Tile::GR, CW = 2 * GR, S4 = Tile::S4, TT = kScanKeep, NT = kBwdWarps * 32, NC = Own::NC, OS = Own::STEPS;
    constexpr bool WHOLE = PASS == SCAN_WHOLE;
    __shared__ __align__(16) Tile sm;
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int grp = lane / LPC, j = lane % LPC;
    const int n = blockIdx.z, span = WHOLE ? blockIdx.y : blockIdx.y + 1;       // nothing in front of the first span asks for its end
    const int per = p.D / p.G, blocks = (per + CW * kBwdWarps - 1) / (CW * kBwdWarps);
    const int g = blockIdx.x / blocks;
    const int ch = ((blockIdx.x % blocks) * kBwdWarps + warp) * CW + 2 * grp;                // inside the group
    const bool on[2] = {ch < per, ch + 1 < per};
    const int last = min(ch, per - (PAIRS ? 2 : 1));        // a lane without a channel reads the last one's rows, counts as steps behind the end, and writes nothing
    const int d[2] = {g * per + last, g * per + min(last + 1, per - 1)};
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
    const int t0 = span * p.span, tend = min(t0 + p.span, p.L), t1 = min(tend, len);
    const bool gated = p.z.p != nullptr;
    const int os = Own::step(j), oc = Own::channel(j);
    const int od[2] = {d[oc], d[1]};                        // the own pairs' channels
    const bool mine[2] = {on[oc] && Own::first(j), on[1] && Own::first(j)};
    const T* x = static_cast<const T*>(p.x.p) + n * p.x.sN;
    const T* dt = static_cast<const T*>(p.dt.p) + n * p.dt.sN;
    const T* z = static_cast<const T*>(p.z.p) + n * p.z.sN;
    const T* gout = static_cast<const T*>(p.gout.p) + n * p.gout.sN;
    T* gx = static_cast<T*>(p.gx.p) + n * p.gx.sN;
    T* gdt = static_cast<T*>(p.gdt.p) + n * p.gdt.sN;
    T* gz = static_cast<T*>(p.gz.p) + n * p.gz.sN;
    auto put = [&](T* row, const float (&v)[NC]) {
        if constexpr (NC == 2) store_two<PAIRS>(row, od, mine, v);
        else if (mine[0]) row[od[0]] = from_f32<T>(v[0]);
    };
    const int row = scan_row(p.S);
    const long long keep_step = (long long)p.D * row;
    const float* keep = p.checkpoints + (long long)n * ((p.L + TT - 1) / TT) * keep_step + 4 * j;
    const bool has = 4 * j < row;

    const long long spans_at = ((long long)n * p.spans + span) * p.D;
    f2 A[2][2], carry[2][2], dA[2][2];
    float bias[NC], skip[NC], gskip[NC], gbias[NC], dsum[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        bias[c] = p.dt_bias ? p.dt_bias[od[c]] : 0.f;
        skip[c] = p.skip ? p.skip[od[c]] : 0.f;
        gskip[c] = gbias[c] = dsum[c] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < 2; c++) {
        float a[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = 4 * j + i < p.S;
            a[i] = in ? rate_of(p.A[(long long)d[c] * p.S + 4 * j + i]) : 0.f;
            s[i] = in && WHOLE && p.spans > 1 ? p.ends[(spans_at + d[c]) * p.S + 4 * j + i] : 0.f;
        }
        A[c][0] = f2_pack(a[0], a[1]); A[c][1] = f2_pack(a[2], a[3]);
        carry[c][0] = f2_pack(s[0], s[1]); carry[c][1] = f2_pack(s[2], s[3]);
        dA[c][0] = dA[c][1] = 0;
        if (WHOLE) sm.dA[warp][c][lane] = make_float4(0.f, 0.f, 0.f, 0.f);
    }

    // the next tile's streams as they are in memory, the state before it, and its rows of B and C
    Raw rx[2][OS], rd[2][OS], rz[2][OS], rg[2][OS];
    float4 rh[2] = {};
    constexpr int BC = (TT * S4 + NT - 1) / NT;
    T rB[BC], rC[BC];
    const int bc_row = threadIdx.x / S4, bc_s = threadIdx.x % S4;
    const bool bc_on = (!RAGGED || bc_s < p.S) && bc_row < TT;
    const T* Bp = static_cast<const T*>(p.B.p) + n * p.B.sN + g * p.B.sH + (bc_on ? bc_s : 0);
    const T* Cp = static_cast<const T*>(p.C.p) + n * p.C.sN + g * p.C.sH + (bc_on ? bc_s : 0);
    auto fetch = [&](int t) {
#pragma unroll
        for (int hh = 0; hh < 2; hh++)
#pragma unroll
            for (int i = 0; i < OS; i++) {
                const int u = min(t + kHalf * hh + os + i, t1 - 1);
                rd[hh][i].load(dt + u * p.dt.sL, od);
                rg[hh][i].load(gout + u * p.gout.sL, od);
                if (WHOLE) rx[hh][i].load(x + u * p.x.sL, od);
                if (gated) rz[hh][i].load(z + u * p.z.sL, od);
            }
        if (WHOLE && has)
#pragma unroll
            for (int c = 0; c < 2; c++) rh[c] = *reinterpret_cast<const float4*>(keep + (t / TT) * keep_step + (long long)d[c] * row);
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int u = min(t + bc_row + i * (NT / S4), t1 - 1);
            if (WHOLE) rB[i] = Bp[u * p.B.sL];
            rC[i] = Cp[u * p.C.sL];
        }
    };
    // the CTA's sums of the tile at t, from buffer `b`
    float* bc = p.bc + (((long long)blockIdx.x * p.N + n) * p.L) * (2 * S4);
    auto flush = [&](int t, int b) {
#pragma unroll
        for (int e = 0; e < (TT * 2 * S4 + NT - 1) / NT; e++) {
            const int q = e * NT + threadIdx.x, r = q / (2 * S4), c = q % (2 * S4);
            if (TT * 2 * S4 < NT && r >= TT) break;
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < kBwdWarps; w++) a += sm.bc[b][w][r][c];
            if (t + r < t1) bc[(long long)(t + r) * (2 * S4) + c] = a;
        }
    };
    const int tiles = t1 > t0 ? (t1 - t0 + TT - 1) / TT : 0;
    if (tiles) fetch(t0 + (tiles - 1) * TT);
    int par = 0;
    for (int b = tiles - 1; b >= 0; b--, par ^= 1) {
        const int t = t0 + b * TT;
        float sig[2][OS][NC], wz[2][OS][NC];        // own pairs: softplus'(dt + bias), gout silu'(z)
        Raw kx[2][OS];
#pragma unroll
        for (int i = 0; i < BC; i++) {
            const int r = bc_row + i * (NT / S4);
            if (TT * S4 >= NT || bc_row < TT) {
                const bool in = bc_on && t + r < t1;
                if (WHOLE) sm.B[par][r][bc_s] = in ? to_f32(rB[i]) : 0.f;
                sm.C[par][r][bc_s] = in ? to_f32(rC[i]) : 0.f;
            }
        }
#pragma unroll
        for (int hh = 0; hh < 2; hh++)
#pragma unroll
            for (int i = 0; i < OS; i++) {
                const int r = kHalf * hh + os + i;
                float dl[NC], dx[NC], gy[NC];
                if (WHOLE) kx[hh][i] = rx[hh][i];
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const bool in = t + r < t1 && on[NC == 2 ? c : oc];
                    const float raw = rd[hh][i].get(c) + bias[c];
                    dl[c] = raw;
                    sig[hh][i][c] = 1.f;
                    if (p.softplus) {
                        dl[c] = softplus_(raw);
                        if (WHOLE) sig[hh][i][c] = sigmoidf_(raw);
                    }
                    dl[c] = in ? dl[c] : 0.f;
                    dx[c] = WHOLE && in ? dl[c] * rx[hh][i].get(c) : 0.f;
                    const float go = in ? rg[hh][i].get(c) : 0.f;
                    gy[c] = go;
                    wz[hh][i][c] = 0.f;
                    if (gated) {
                        const float zz = rz[hh][i].get(c), s = sigmoidf_(zz);
                        gy[c] = in ? go * silu_of(zz, s) : 0.f;
                        wz[hh][i][c] = go * silu_grad_of(zz, s);
                    }
                    if (!WHOLE && Own::first(j)) dsum[c] += dl[c];
                }
                if constexpr (NC == 2) {
                    sm.st[warp][r][grp] = make_float4(dl[0], dx[0], dl[1], dx[1]);
                    sm.gy[warp][r][grp] = make_float2(gy[0], gy[1]);
                } else if (Own::first(j)) {
                    reinterpret_cast<float2*>(&sm.st[warp][r][grp])[oc] = make_float2(dl[0], dx[0]);
                    reinterpret_cast<float*>(&sm.gy[warp][r][grp])[oc] = gy[0];
                }
            }
        const f2 h0[2][2] = {{f2_pack(rh[0].x, rh[0].y), f2_pack(rh[0].z, rh[0].w)}, {f2_pack(rh[1].x, rh[1].y), f2_pack(rh[1].z, rh[1].w)}};
        __syncthreads();
        if (WHOLE && b < tiles - 1) flush(t + TT, par ^ 1);
        if (b > 0) fetch(t - TT);
        if (!WHOLE) {
#pragma unroll
            for (int r = TT - 1; r >= 0; r--) {
                const float4 s = sm.st[warp][r][grp];
                const float2 gy = sm.gy[warp][r][grp];
                const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][r][4 * j]);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float dl = c ? s.z : s.x, gg = c ? gy.y : gy.x;
                    const f2 d2 = f2_pack(dl, dl), gy2 = f2_pack(gg, gg);
                    carry[c][0] = fmul2(decay_pair(d2, A[c][0]), ffma2(cc.x, gy2, carry[c][0]));
                    carry[c][1] = fmul2(decay_pair(d2, A[c][1]), ffma2(cc.y, gy2, carry[c][1]));
                    if (RAGGED) keep_states(carry[c], 4 * j, p.S);
                }
            }
            __syncwarp();
            continue;
        }
        auto advance = [&](f2 (&h)[2], int c, int r, f2& e0, f2& e1, float dl, float dx, const ulonglong2& bb) {
            const f2 d2 = f2_pack(dl, dl), x2 = f2_pack(dx, dx);
            e0 = decay_pair(d2, A[c][0]);
            e1 = decay_pair(d2, A[c][1]);
            h[0] = ffma2(e0, h[0], fmul2(x2, bb.x));
            h[1] = ffma2(e1, h[1], fmul2(x2, bb.y));
            if (RAGGED) keep_states(h, 4 * j, p.S);
        };
        f2 mid[2][2] = {{h0[0][0], h0[0][1]}, {h0[1][0], h0[1][1]}};
#pragma unroll
        for (int r = 0; r < kHalf; r++) {
            const float4 s = sm.st[warp][r][grp];
            const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B[par][r][4 * j]);
            f2 e0, e1;
            advance(mid[0], 0, r, e0, e1, s.x, s.y, bb);
            advance(mid[1], 1, r, e0, e1, s.z, s.w, bb);
        }
#pragma unroll
        for (int hh = 1; hh >= 0; hh--) {
            f2 a[kHalf][2][2], H[kHalf][2][2], h[2][2];
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < 2; i++) h[c][i] = hh ? mid[c][i] : h0[c][i];
            float v[2 * kHalf], q[2 * kHalf];
#pragma unroll
            for (int r = 0; r < kHalf; r++) {
                const float4 s = sm.st[warp][kHalf * hh + r][grp];
                const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B[par][kHalf * hh + r][4 * j]);
                ulonglong2 cc = {};
                if (gated) cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][kHalf * hh + r][4 * j]);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    advance(h[c], c, r, a[r][c][0], a[r][c][1], c ? s.z : s.x, c ? s.w : s.y, bb);
                    H[r][c][0] = h[c][0];
                    H[r][c][1] = h[c][1];
                    if (gated) v[2 * r + c] = f2_hsum(ffma2(cc.y, h[c][1], fmul2(cc.x, h[c][0])));
                }
            }
            if (gated) {
                sum_lanes<2 * kHalf, LPC, 1>(v, lane);
#pragma unroll
                for (int i = 0; i < OS; i++) {
                    const int u = t + kHalf * hh + os + i;
                    float w[NC];
#pragma unroll
                    for (int c = 0; c < NC; c++) w[c] = wz[hh][i][c] * fmaf(skip[c], kx[hh][i].get(c), v[i * NC + c]);
                    if (u < t1) put(gz + u * p.gz.sL, w);
                }
            }
            f2 part[2][2] = {};             // of dA: over four steps first, so that long sequences lose no small terms
#pragma unroll
            for (int r = kHalf - 1; r >= 0; r--) {
                const float4 s = sm.st[warp][kHalf * hh + r][grp];
                const float2 gy = sm.gy[warp][kHalf * hh + r][grp];
                const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C[par][kHalf * hh + r][4 * j]);
                const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B[par][kHalf * hh + r][4 * j]);
                f2 gB0, gB1, gC0, gC1;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float dl = c ? s.z : s.x, dx = c ? s.w : s.y, gyc = c ? gy.y : gy.x;
                    const f2 d2 = f2_pack(dl, dl), x2 = f2_pack(dx, dx), gy2 = f2_pack(gyc, gyc);
                    f2 gg[2] = {ffma2(cc.x, gy2, carry[c][0]), ffma2(cc.y, gy2, carry[c][1])};
                    if (RAGGED) keep_states(gg, 4 * j, p.S);
                    carry[c][0] = fmul2(a[r][c][0], gg[0]);
                    carry[c][1] = fmul2(a[r][c][1], gg[1]);
                    if (RAGGED) keep_states(carry[c], 4 * j, p.S);
                    const f2 b0 = r ? H[r ? r - 1 : 0][c][0] : hh ? mid[c][0] : h0[c][0], b1 = r ? H[r ? r - 1 : 0][c][1] : hh ? mid[c][1] : h0[c][1];
                    const f2 e0 = fmul2(carry[c][0], b0), e1 = fmul2(carry[c][1], b1);
                    v[2 * r + c] = f2_hsum(ffma2(gg[1], bb.y, fmul2(gg[0], bb.x)));
                    q[2 * r + c] = f2_hsum(ffma2(e1, A[c][1], fmul2(e0, A[c][0])));
                    part[c][0] = ffma2(e0, d2, part[c][0]);
                    part[c][1] = ffma2(e1, d2, part[c][1]);
                    gB0 = c ? ffma2(gg[0], x2, gB0) : fmul2(gg[0], x2); gB1 = c ? ffma2(gg[1], x2, gB1) : fmul2(gg[1], x2);
                    gC0 = c ? ffma2(gy2, H[r][c][0], gC0) : fmul2(gy2, H[r][c][0]); gC1 = c ? ffma2(gy2, H[r][c][1], gC1) : fmul2(gy2, H[r][c][1]);
                }
                float w[8];
                f2_unpack(gB0, w[0], w[1]);
                f2_unpack(gB1, w[2], w[3]);
                f2_unpack(gC0, w[4], w[5]);
                f2_unpack(gC1, w[6], w[7]);
                sum_lanes<8, GR, LPC>(w, lane);
                float* to = sm.bc[par][warp][kHalf * hh + r];
                if constexpr (GR <= 8) {
                    constexpr int NV = 8 / GR;
#pragma unroll
                    for (int i = 0; i < NV; i++) {
                        const int k = grp * NV + i;
                        to[(k >> 2) * S4 + 4 * j + (k & 3)] = w[i];
                    }
                } else {
                    constexpr int SH = GR / 8;
                    const int k = grp / SH;
                    if (grp % SH == 0) to[(k >> 2) * S4 + 4 * j + (k & 3)] = w[0];
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < 2; i++) dA[c][i] = fadd2(dA[c][i], part[c][i]);
            sum_lanes<2 * kHalf, LPC, 1>(v, lane);
            sum_lanes<2 * kHalf, LPC, 1>(q, lane);
#pragma unroll
            for (int i = 0; i < OS; i++) {
                const int r = kHalf * hh + os + i, u = t + r;
                float wx[NC], wd[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const float xx = kx[hh][i].get(c);
                    const float dl = NC == 2 ? (c ? sm.st[warp][r][grp].z : sm.st[warp][r][grp].x) : (oc ? sm.st[warp][r][grp].z : sm.st[warp][r][grp].x);
                    const float gy = NC == 2 ? (c ? sm.gy[warp][r][grp].y : sm.gy[warp][r][grp].x) : (oc ? sm.gy[warp][r][grp].y : sm.gy[warp][r][grp].x);
                    wx[c] = fmaf(dl, v[i * NC + c], skip[c] * gy);
                    wd[c] = fmaf(xx, v[i * NC + c], q[i * NC + c] * kLn2) * sig[hh][i][c];
                    if (u < t1) {
                        gskip[c] = fmaf(gy, xx, gskip[c]);
                        gbias[c] += wd[c];
                    }
                }
                if (u < t1) {
                    put(gx + u * p.gx.sL, wx);
                    put(gdt + u * p.gdt.sL, wd);
                }
            }
        }
        __syncwarp();           // the warp's st and gy are read
        // gA is a sum over all steps of terms of either sign: four steps, then sixteen tiles, then the rest, so that its error stays
        // that of the states it is made of
        if (b % 16 == 0)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float4 s = sm.dA[warp][c][lane];
                float v[4];
                f2_unpack(dA[c][0], v[0], v[1]);
                f2_unpack(dA[c][1], v[2], v[3]);
                s.x += v[0]; s.y += v[1]; s.z += v[2]; s.w += v[3];
                sm.dA[warp][c][lane] = s;
                dA[c][0] = dA[c][1] = 0;
            }
    }
    // sums over the lanes that share a channel
#pragma unroll
    for (int c = 0; c < NC; c++) {
        if (!Own::first(j)) gskip[c] = gbias[c] = dsum[c] = 0.f;
#pragma unroll
        for (int o = 1; o < LPC; o <<= 1) {
            if (LPC == 8 && o == 1) continue;       // neighbours hold the other channel
            if (LPC == 16 && o == 2) continue;
            gskip[c] += __shfl_xor_sync(0xffffffffu, gskip[c], o);
            gbias[c] += __shfl_xor_sync(0xffffffffu, gbias[c], o);
            dsum[c] += __shfl_xor_sync(0xffffffffu, dsum[c], o);
        }
    }
    const bool writes[2] = {on[oc] && Own::first(j) && os == 0, on[1] && os == 0};
    if (WHOLE) {
        __syncthreads();
        if (tiles) flush(t0, par ^ 1);
        const float zero[NC] = {};
        for (int u = max(t0, t1) + os; u < tend; u += kHalf) {
            const int most = min(u + OS, tend);
            for (int w = u; w < most; w++) {
                put(gx + w * p.gx.sL, zero);
                put(gdt + w * p.gdt.sL, zero);
                if (gated) put(gz + w * p.gz.sL, zero);
            }
        }
        float* sums = p.sums + ((long long)n * p.spans + span) * p.D * (p.S + 2);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float4 s = sm.dA[warp][c][lane];          // the lane's own: the first tile has added the rest
            const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (on[c] && 4 * j + i < p.S) sums[(long long)d[c] * p.S + 4 * j + i] = v[i];
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (writes[c]) {
                sums[(long long)p.D * p.S + od[c]] = gskip[c];
                sums[(long long)p.D * (p.S + 1) + od[c]] = gbias[c];
            }
    } else {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float v[4];
            f2_unpack(carry[c][0], v[0], v[1]);
            f2_unpack(carry[c][1], v[2], v[3]);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (on[c] && 4 * j + i < p.S) p.ends[(spans_at + d[c]) * p.S + 4 * j + i] = v[i];
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (writes[c]) p.dsums[spans_at + od[c]] = dsum[c];
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
    const int lpc = scan_lanes(S), w = kBwdWarps, cw = 64 / lpc, per = D / G;
    const long long sms = sm_count() > 0 ? sm_count() : 148;
    ScanBwdPlan q;
    q.blocks = (int)ceil_div(per, cw * w);
    const long long ctas = (long long)N * G * q.blocks;
    const int forced = tune_get(T_SCAN_CHUNK, 0);
    int spans = 1;
    if (forced > 0) spans = (int)ceil_div(L, ceil_div(forced, kScanKeep) * kScanKeep);
    else if (ctas <= sms) spans = (int)(sms * 2 / ctas);
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

template <typename T, int LPC, bool RAGGED, bool PAIRS>
static int scan_bwd_launch(const ScanParams& p, const ScanBwdPlan& q, cudaStream_t st) {
    const unsigned gx = (unsigned)(p.G * q.blocks);
    constexpr int threads = kBwdWarps * 32;
    if (q.spans > 1) {
        if (int rc = launch_dependent(scan_bwd_kernel<T, LPC, RAGGED, PAIRS, SCAN_ENDS>, p, dim3(gx, q.spans - 1, p.N), threads, 0, st, nullptr)) return rc;
        if (int rc = launch_scan_join(p, true, st)) return rc;
    }
    return launch_dependent(scan_bwd_kernel<T, LPC, RAGGED, PAIRS, SCAN_WHOLE>, p, dim3(gx, q.spans, p.N), threads, 0, st, "scan_bwd_kernel");
}
template <typename T>
static int scan_bwd_dispatch(const ScanParams& p, const ScanBwdPlan& q, cudaStream_t st) {
    const int lpc = scan_lanes(p.S);
    const bool ragged = p.S != 4 * lpc;
#define FWP_SCAN_BWD(LPC) (ragged ? scan_bwd_launch<T, LPC, true, false>(p, q, st) : p.pairs ? scan_bwd_launch<T, LPC, false, true>(p, q, st) : scan_bwd_launch<T, LPC, false, false>(p, q, st))
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
    p.pairs = D / G % 2 == 0;
    for (const Stream* s : {&p.x, &p.dt, &p.z, &p.gout, &p.gx, &p.gdt, &p.gz}) p.pairs = p.pairs && rows_aligned(*s, esz, 2 * esz);
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
