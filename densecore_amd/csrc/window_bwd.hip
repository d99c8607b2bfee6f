// Backward of attention with a sliding window and sinks (window.hpp): with P = exp(scale q k^T - lse) at
// the visible pairs, dsum = rowsum(dO * O) and dS = P (dO v^T - dsum),
//     dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,
// dK and dV summed over the query heads that share a kv head.  Two kernels, no atomics:
//   * window_dq_kernel (queries stay, the forward's structure) also forms dsum;
//   * window_dkdv_kernel (keys stay): a workgroup owns 128 keys, 32 per wave, and walks the queries that see one
//     of them, head after head; where its tiles fill the LDS, eight waves halve each step's queries and join at the end.
// Bound: as the forward, a wave's own chain at two waves to a SIMD.  B2 H32/8 L8192 E128 W1024 with 4 sinks bf16:
// dQ 599 us (650 TFLOP/s of the visible pairs' three products, 860 with dS's lo terms; MFMA busy 45%), dK and dV 1016 us
// (510 of four products, 760 with lo terms; 38%), the sinks' pieces joined in 11.  Float32 B8 H12 L1024 E64 W256: 99,
// 141 and 9 us.
// Rows whose result is not finite are computed again in plain float32 over their visible pairs (as in
// the forward, matrix products spread NaN and infinities to rows that do not see them).
#include <algorithm>

#include "params.hpp"
#include "window.hpp"

namespace dc {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kM = 32 * kWaves;
template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // dQ: keys per tile
// Two waves per SIMD or more, but for float32 at D = 128 (three parts of two operands and the sums take 350 registers).
template <typename T, int D>
constexpr int kWavesPerSimd = sizeof(T) == 2 || D <= 64 ? 2 : 1;
// dK / dV: with two halves, waves w and w + 4 own the same 32 keys and halve each step's queries, one workgroup to a
// CU (its tiles fill the LDS); with one, several workgroups share a CU and a wave has twice the products between two
// barriers: B4 H32 L4096 W1024 bf16 E64 backward 884 us with halves, 765 without, E32 565 and 444 (three waves per SIMD);
// float32 E32 433 and 390, while at E64 keeping V in registers for it spills (239 and 256).
template <typename T, int D>
constexpr int kHalves = D == 32 || (sizeof(T) == 2 && D == 64) ? 1 : kWavesPerSimd<T, D>;
template <typename T, int D>
constexpr int kQueries = sizeof(T) == 2 || D <= 64 ? 64 : 32;  // per step
// dK / dV: K's, V's operands in LDS and not in registers, where these would spill (at D = 128 the sums alone
// take half of bf16's, and float32's take 350 with one wave per SIMD).
template <typename T, int D>
constexpr bool kKLds = sizeof(T) == 2 && D == 128;
template <typename T, int D>
constexpr bool kVLds = D >= 64 && (sizeof(T) == 2 ? D == 128 : D == 64);

template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D>))) void window_dq_kernel(WinArgs a) {
    typedef Ops<T> O;
    constexpr int BN = kKeys<T>, NT = BN / 32, KSTEP = D / 16, NDT = D / 32;
    typedef Stage<T, BN, D, kThreads, VEC> St;
    __shared__ typename St::Tile sk[2], sv[2];
    static_assert(!kTurned<T, D, VEC> || sizeof(sk) >= kWaves * kRoom<D> * sizeof(u32x4), "the results' turn");

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nqt = (a.L + kM - 1) / kM;
    const int w = logical_block();
    // (The heads of a kv head side by side, as in the forward.)
    const int qt = nqt - 1 - w / a.repeat % nqt, kvh = w / a.repeat / nqt;
    const int b = kvh / a.Hkv, hk = kvh % a.Hkv, h = hk * a.repeat + w % a.repeat, bh = b * a.H + h;
    const int r0 = qt * kM, wr0 = r0 + 32 * wave, r = wr0 + lr;
    const bool in = r < a.L;
    const int l = in ? r : a.L - 1, p = in ? a.offset + l : -1;
    const int64_t row = (int64_t)bh * a.L + l;
    const int wp0 = a.offset + wr0, wp1 = a.offset + min(wr0 + 31, a.L - 1);  // wp1 < wp0: no rows
    const Band band = band_of(a.offset + r0, a.offset + min(r0 + kM, a.L) - 1, a.S, a.window, a.sinks, BN);

    const T *kb = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T *vb = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const T *qb = static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[1];
    const T *gb = static_cast<const T *>(a.dout) + b * a.gs[0] + h * a.gs[1];
    const T *ob = static_cast<const T *>(a.out_in) + (int64_t)bh * a.L * a.E;
    const T *rb = static_cast<const T *>(a.rest) + (int64_t)bh * a.L * a.E;

    const uint32_t rowb = row_lanebase<BN, D>(lane), trb = tr_lanebase<BN, D>(lane);
    St kst, vst;
    auto start = [&](int i) {
        const int n0 = band.tile(i) * BN, nr = min(BN, a.S - n0);
        kst.start(sk[i & 1], kb + (int64_t)n0 * a.ks[2], a.ks[2], nr, a.E, tid);
        vst.start(sv[i & 1], vb + (int64_t)n0 * a.vs[2], a.vs[2], nr, a.E, tid);
    };
    auto finish = [&](int i) {
        kst.finish(sk[i & 1], tid);
        vst.finish(sv[i & 1], tid);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) St::clear(sk[i], a.E, tid), St::clear(sv[i], a.E, tid);
    if (band.n > 0) start(0);  // on its way while the queries load

    typename O::Frag qf[KSTEP], gf[KSTEP];
    float dsum = 0.f;
#pragma unroll
    for (int t = 0; t < KSTEP; ++t) {
        qf[t] = O::template load<VEC>(qb + l * a.qs[2], 16 * t + 8 * g, a.E, in);
        gf[t] = O::template load<VEC>(gb + l * a.gs[2], 16 * t + 8 * g, a.E, in);
        dsum += O::dot(gf[t], O::template load<VEC>(ob + (int64_t)l * a.E, 16 * t + 8 * g, a.E, in));
        if (sizeof(T) == 2 && a.rest) dsum += O::dot(gf[t], O::template load<VEC>(rb + (int64_t)l * a.E, 16 * t + 8 * g, a.E, in));
    }
    dsum = xor32_add(dsum);
    if (in && g == 0) a.dsum[row] = dsum;
    const float nlse = in ? -a.lse_in[row] * kLog2e : 0.f;

    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;

    if (band.n > 0) finish(0);

    auto step = [&](int i) {
        const int n0 = band.tile(i) * BN;
        const bool all = n0 + BN <= a.S && n0 + BN - 1 <= wp0 && (wp1 - n0 < a.window || n0 + BN <= a.sinks);
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            const int k0 = n0 + 32 * kt;
            if (!(wp0 <= wp1 && k0 < a.S && k0 <= wp1 && (wp0 - (k0 + 31) < a.window || k0 < a.sinks))) continue;
            f32x16 s, t;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.f, t[e] = -dsum;
#pragma unroll
            for (int st = 0; st < KSTEP; ++st) {
                s = O::mma(O::row(sk[i & 1], rowb, 32 * kt, st), qf[st], s);
                t = O::mma(O::row(sv[i & 1], rowb, 32 * kt, st), gf[st], t);
            }
            reads_ahead<2 * KSTEP, O::MMAS, O::READS, sizeof(T) == 2 ? 4 : 2>();
            pin(s), pin(t);
            __builtin_amdgcn_sched_barrier(0);
            typename O::Frag kf[2][NDT];  // K^T of the 16-key halves, the first while dS is formed
            auto load_k = [&](int u) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) kf[u][dt] = O::tr(sk[i & 1], trb, 32 * kt + 16 * u, dt);
            };
            load_k(0);
            if (all) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = exp2_fast(fmaf(s[e], a.scale_log2, nlse));
            } else {
                const SeenKeys seen(p, k0 + 4 * g, a.S, a.window, a.sinks);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = exp2_fast(seen(acc_const(e)) ? fmaf(s[e], a.scale_log2, nlse) : -INFINITY);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= t[e];
            if (sizeof(T) == 2) load_k(1);
            O::mma_p(kf[0], s, 0, acc);
            if (sizeof(T) != 2) load_k(1);
            O::mma_p(kf[1], s, 8, acc);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) pin(acc[dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int i = 0; i < band.n; ++i) {
        __syncthreads();
        if (i + 1 < band.n) start(i + 1);
        step(i);
        if (i + 1 < band.n) finish(i + 1);
    }

    float test = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) test += not_finite(acc[dt]);
    const uint64_t wrong = __ballot(in && test != 0.f);
    uint32_t again = (uint32_t)wrong | (uint32_t)(wrong >> 32);
    T *dq = static_cast<T *>(a.dq);
    if constexpr (kTurned<T, D, VEC>) {
        __syncthreads();  // everyone is done with the tiles, which the results now pass through
        store_turned<D>(reinterpret_cast<u32x4 *>(sk) + wave * kRoom<D>, lane, a.E,
                        [&](int dt, int e) { return acc[dt][e] * a.scale; }, [&](int r1) -> __bf16 * {
                            return wr0 + r1 < a.L && !((again >> r1) & 1) ? dq + ((int64_t)bh * a.L + wr0 + r1) * a.E : nullptr;
                        });
    } else if (in && !((again >> lr) & 1)) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                store4<T, VEC>(dq + row * a.E, dt * 32 + acc_row(e, g), a.E, acc[dt][e] * a.scale, acc[dt][e + 1] * a.scale,
                               acc[dt][e + 2] * a.scale, acc[dt][e + 3] * a.scale);
    }
    // Rows again: lanes are keys for dS and dims for the sum.
    for (; again; again &= again - 1) {
        const int rl = wr0 + __builtin_ctz(again), rp = a.offset + rl;
        const int64_t rr = (int64_t)bh * a.L + rl;
        const T *q1 = qb + rl * a.qs[2], *g1 = gb + rl * a.gs[2];
        float rs = plain_dot<T>(g1, ob + (int64_t)rl * a.E, a.E);
        if (sizeof(T) == 2 && a.rest) rs += plain_dot<T>(g1, rb + (int64_t)rl * a.E, a.E);
        const float rlse = a.lse_in[rr];
        if (lane == 0) a.dsum[rr] = rs;
        float o[2] = {0.f, 0.f};
        // (The same in all lanes.)  A NaN lse or dsum is in every dS of the row.
        const bool lost = (rlse != rlse || rs != rs) && sees_any(a, rp);
        if (lost) o[0] = o[1] = NAN;
        for (int i = 0; i < band.n && !lost; ++i) {
            const int n0 = band.tile(i) * BN, key = n0 + lane;
            const bool ok = lane < BN && key < a.S && sees(rp, key, a.window, a.sinks);
            float ds = 0.f;
            if (ok) {
                const float pr = exp2_fast((plain_dot<T>(q1, kb + key * a.ks[2], a.E) * a.scale - rlse) * kLog2e);
                ds = pr * (plain_dot<T>(g1, vb + key * a.vs[2], a.E) - rs);
            }
            for (uint64_t left = __ballot(ok); left; left &= left - 1) {
                const int j = __builtin_ctzll(left);
                const float dj = __shfl(ds, j, 64);
                const T *k1 = kb + (n0 + j) * a.ks[2];
                if (lane < a.E) o[0] = fmaf(dj, to_f32<T>(k1[lane]), o[0]);
                if (lane + 64 < a.E) o[1] = fmaf(dj, to_f32<T>(k1[lane + 64]), o[1]);
            }
            if (all_nan(lane, a.E, o[0], o[1])) break;
        }
        if (lane < a.E) dq[rr * a.E + lane] = from_f32<T>(o[0] * a.scale);
        if (lane + 64 < a.E) dq[rr * a.E + lane + 64] = from_f32<T>(o[1] * a.scale);
    }
}

// The queries [l0, l1) of a head that see one of the keys n0 .. n1 - 1.
__host__ __device__ inline void query_range(const WinArgs &a, int n0, int n1, int &l0, int &l1) {
    l0 = n0 > a.offset ? n0 - a.offset : 0;
    const int64_t end = (int64_t)n1 - 1 + a.window - a.offset;
    l1 = n0 < a.sinks || end > a.L ? a.L : (int)end;
    if (l0 > a.L) l0 = a.L;
    if (l1 < l0) l1 = l0;
}

// Steps (of QM queries, over the heads that share the kv head) of the key tile at n0.
__host__ __device__ inline int64_t tile_steps(const WinArgs &a, int n0, int QM) {
    int l0, l1;
    query_range(a, n0, n0 + kM < a.S ? n0 + kM : a.S, l0, l1);
    return (int64_t)((l1 - l0 + QM - 1) / QM) * a.repeat;
}

// Key tile kt's pieces and the first one's slot in kv_part (a slot: kM keys of dK, then of dV).
struct Pieces {
    int n;
    int64_t slot;
};
DEVI Pieces pieces_of(const WinArgs &a, int nkt, int bhk, int kt) {
    const int64_t head = (int64_t)a.sink_tiles * a.sink_pieces + (int64_t)(nkt - a.sink_tiles) * a.tile_pieces;
    if (kt < a.sink_tiles) return {a.sink_pieces, bhk * head + (int64_t)kt * a.sink_pieces};
    return {a.tile_pieces, bhk * head + (int64_t)a.sink_tiles * a.sink_pieces + (int64_t)(kt - a.sink_tiles) * a.tile_pieces};
}

template <typename T, int D, bool VEC>
__global__ __launch_bounds__((kThreads * kHalves<T, D>))
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D>))) void window_dkdv_kernel(WinArgs a) {
    typedef Ops<T> O;
    constexpr int HALVES = kHalves<T, D>, QM = kQueries<T, D>, THREADS = kThreads * HALVES, KSTEP = D / 16, NDT = D / 32;
    constexpr bool KLDS = kKLds<T, D>, VLDS = kVLds<T, D>;
    typedef Stage<T, QM, D, THREADS, VEC> St;
    typedef Stage<T, VLDS ? kM : 32, D, THREADS, VEC> StV;
    struct Main {
        typename St::Tile q[2], g[2];
        float lse[2][QM], dsum[2][QM];  // -lse log2 e (-inf behind the last row: P = 0) and -dsum
        typename StV::Tile k[KLDS ? 1 : 0], v[VLDS ? 1 : 0];
    };
    union Smem {
        Main m;
        float red[HALVES > 1][kWaves][NDT][16][64];  // the second half's sums on their way to the first
    };
    __shared__ Smem sm;

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave % kWaves, half = wave / kWaves;
    const int nkt = (a.S + kM - 1) / kM;
    const int per = a.sink_tiles * a.sink_pieces + (nkt - a.sink_tiles) * a.tile_pieces;  // blocks of a kv head
    const int w = logical_block(), bhk = w / per;
    int kt = w % per, piece;
    if (kt < a.sink_tiles * a.sink_pieces) {
        piece = kt % a.sink_pieces, kt = kt / a.sink_pieces;
    } else {
        kt -= a.sink_tiles * a.sink_pieces;
        piece = kt % a.tile_pieces, kt = a.sink_tiles + kt / a.tile_pieces;
    }
    const Pieces pcs = pieces_of(a, nkt, bhk, kt);
    const int n0 = kt * kM, b = bhk / a.Hkv, hk = bhk % a.Hkv;
    const int kw0 = n0 + 32 * kw, key = kw0 + lr;
    const T *kb = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T *vb = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const T *qb = static_cast<const T *>(a.q) + b * a.qs[0];
    const T *gb = static_cast<const T *>(a.dout) + b * a.gs[0];
    int l0, l1;
    query_range(a, n0, min(n0 + kM, a.S), l0, l1);
    const int per_head = (l1 - l0 + QM - 1) / QM;
    const int64_t all_steps = (int64_t)per_head * a.repeat;
    const int i0 = (int)(piece * all_steps / pcs.n), i1 = (int)((piece + 1) * all_steps / pcs.n);

    St qst, gst;
    float stat = 0.f;
    // Step i's head and first query; at(i + 1) is at(i) moved on.
    struct At {
        int h, m;
    };
    auto first = [&](int i) { return At{hk * a.repeat + i / per_head, l0 + i % per_head * QM}; };
    auto next = [&](At x) { return x.m + QM < l1 ? At{x.h, x.m + QM} : At{x.h + 1, l0}; };
    auto start = [&](int i, At x) {
        const int h = x.h, m0 = x.m, nr = min(QM, a.L - m0);
        qst.start(sm.m.q[i & 1], qb + h * a.qs[1] + m0 * a.qs[2], a.qs[2], nr, a.E, tid);
        gst.start(sm.m.g[i & 1], gb + h * a.gs[1] + m0 * a.gs[2], a.gs[2], nr, a.E, tid);
        // (As it lies: arithmetic on it here would wait for every transfer issued so far.)
        if (tid < 2 * QM) stat = (tid < QM ? a.lse_in : a.dsum)[((int64_t)b * a.H + h) * a.L + m0 + min(tid % QM, nr - 1)];
    };
    auto finish = [&](int i, At x) {
        qst.finish(sm.m.q[i & 1], tid);
        gst.finish(sm.m.g[i & 1], tid);
        if (tid < QM) sm.m.lse[i & 1][tid] = x.m + tid < a.L ? -stat * kLog2e : -INFINITY;
        else if (tid < 2 * QM) sm.m.dsum[i & 1][tid - QM] = x.m + tid - QM < a.L ? -stat : 0.f;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) St::clear(sm.m.q[i], a.E, tid), St::clear(sm.m.g[i], a.E, tid);
    auto hold = [&](StV &x, auto &tile, const T *src, int64_t ld) {
        StV::clear(tile, a.E, tid);
        x.start(tile, src + n0 * ld, ld, min(kM, a.S - n0), a.E, tid);
    };
    StV kst, vst;
    if constexpr (KLDS) hold(kst, sm.m.k[0], kb, a.ks[2]);
    if constexpr (VLDS) hold(vst, sm.m.v[0], vb, a.vs[2]);
    if constexpr (KLDS) kst.finish(sm.m.k[0], tid);
    if constexpr (VLDS) vst.finish(sm.m.v[0], tid);
    At now = {0, 0};
    if (i0 < i1) now = first(i0), start(i0, now);

    typename O::Frag kf[KLDS ? 1 : KSTEP], vf[VLDS ? 1 : KSTEP];
#pragma unroll
    for (int t = 0; t < KSTEP; ++t) {
        const int kr = min(key, a.S - 1);
        if constexpr (!KLDS) kf[t] = O::template load<VEC>(kb + kr * a.ks[2], 16 * t + 8 * g, a.E, key < a.S);
        if constexpr (!VLDS) vf[t] = O::template load<VEC>(vb + kr * a.vs[2], 16 * t + 8 * g, a.E, key < a.S);
    }
    if (i0 < i1) finish(i0, now);
    f32x16 dk[NDT], dv[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.f;
    const uint32_t rowb = row_lanebase<QM, D>(lane), trb = tr_lanebase<QM, D>(lane);
    const uint32_t rowk = row_lanebase<VLDS ? kM : 32, D>(lane);

    auto step = [&](int i, At x, int part) {
        const int buf = i & 1, mq = x.m + 32 * part, r0 = 32 * part;
        const int q0 = a.offset + mq, q1 = a.offset + min(mq + 31, a.L - 1);
        if (mq >= a.L || kw0 >= a.S || kw0 > q1 || (q0 - (kw0 + 31) >= a.window && kw0 >= a.sinks)) return;
        const bool all = kw0 + 31 < a.S && kw0 + 31 <= q0 && (q1 - kw0 < a.window || kw0 + 31 < a.sinks);
        f32x16 s, t;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 nd = *reinterpret_cast<const f32x4 *>(&sm.m.dsum[buf][r0 + 8 * r4 + 4 * g]);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * r4 + j] = 0.f, t[4 * r4 + j] = nd[j];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < KSTEP; ++st) {
            if constexpr (KLDS) s = O::mma(O::row(sm.m.q[buf], rowb, r0, st), O::row(sm.m.k[0], rowk, 32 * kw, st), s);
            else s = O::mma(O::row(sm.m.q[buf], rowb, r0, st), kf[st], s);
            if constexpr (VLDS) t = O::mma(O::row(sm.m.g[buf], rowb, r0, st), O::row(sm.m.v[0], rowk, 32 * kw, st), t);
            else t = O::mma(O::row(sm.m.g[buf], rowb, r0, st), vf[st], t);
        }
        reads_ahead<KSTEP, 2 * O::MMAS, (2 + KLDS + VLDS) * O::READS, sizeof(T) == 2 ? 2 : 1>();
        pin(s), pin(t);
        __builtin_amdgcn_sched_barrier(0);
        // dV^T += dO^T P and dK^T += Q^T dS, 16 queries at a time; bf16's transposed operands are read a
        // product ahead, the first while P and dS are formed.
        constexpr int FB = sizeof(T) == 2 ? 2 : 1;
        typename O::Frag f[FB][NDT];
        auto load = [&](int n) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                f[n % FB][dt] = O::tr((n & 1) ? sm.m.q[buf] : sm.m.g[buf], trb, r0 + 16 * (n >> 1), dt);
        };
        f32x4 nl[4];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) nl[r4] = *reinterpret_cast<const f32x4 *>(&sm.m.lse[buf][r0 + 8 * r4 + 4 * g]);
        load(0);
        if (all) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = exp2_fast(fmaf(s[e], a.scale_log2, nl[e >> 2][e & 3]));
                t[e] *= s[e];
            }
        } else {
            const SeenBy seen(key, q0 + 4 * g, a.S, a.window, a.sinks);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = exp2_fast(seen(acc_const(e)) ? fmaf(s[e], a.scale_log2, nl[e >> 2][e & 3]) : -INFINITY);
                t[e] *= s[e];
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (sizeof(T) == 2 && n + 1 < 4) load(n + 1);
            if (n & 1) O::mma_p(f[n % FB], t, 8 * (n >> 1), dk);
            else O::mma_p(f[n % FB], s, 8 * (n >> 1), dv);
            if (sizeof(T) != 2 && n + 1 < 4) load(n + 1);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) pin((n & 1) ? dk[dt] : dv[dt]);
            __builtin_amdgcn_sched_barrier(0);  // or all four reads are issued at once, into spilled registers
        }
    };
    for (int i = i0; i < i1; ++i) {
        __syncthreads();
        const At then = next(now);
        if (i + 1 < i1) start(i + 1, then);
        if constexpr (32 * HALVES == QM) {
            step(i, now, half);
        } else {
#pragma unroll 1
            for (int part = 0; part < QM / 32; ++part) step(i, now, part);
        }
        if (i + 1 < i1) finish(i + 1, then);
        now = then;
    }

    if constexpr (HALVES == 2) {  // the second half's sums join the first's, dK then dV through the same room
        auto join = [&](f32x16 (&x)[NDT]) {
            __syncthreads();
            if (half == 1) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sm.red[0][kw][dt][e][lane] = x[dt][e];
            }
            __syncthreads();
            if (half == 0) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[dt][e] += sm.red[0][kw][dt][e][lane];
            }
        };
        join(dk), join(dv);
        if (half == 1) return;
    }
    float testk = 0.f, testv = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) testk += not_finite(dk[dt]), testv += not_finite(dv[dt]);
    const uint64_t wrongk = __ballot(key < a.S && testk != 0.f), wrongv = __ballot(key < a.S && testv != 0.f);
    const uint32_t againk = (uint32_t)wrongk | (uint32_t)(wrongk >> 32), againv = (uint32_t)wrongv | (uint32_t)(wrongv >> 32);
    // Rows of this block: results, or its piece's float32 slot.
    T *dko = static_cast<T *>(a.dk) + ((int64_t)bhk * a.S + n0) * a.E, *dvo = static_cast<T *>(a.dv) + ((int64_t)bhk * a.S + n0) * a.E;
    float *pk = a.kv_part + (pcs.slot + piece) * 2 * kM * a.E, *pv = pk + (int64_t)kM * a.E;
    const int at = 32 * kw + lr;
    auto put = [&](const f32x16 (&x)[NDT], float scale, T *out, float *part) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = dt * 32 + acc_row(e, g);
                const float x0 = x[dt][e] * scale, x1 = x[dt][e + 1] * scale, x2 = x[dt][e + 2] * scale, x3 = x[dt][e + 3] * scale;
                if (pcs.n > 1) store4<float, VEC>(part + at * a.E, d, a.E, x0, x1, x2, x3);
                else store4<T, VEC>(out + (int64_t)at * a.E, d, a.E, x0, x1, x2, x3);
            }
    };
    if (key < a.S && !((againk >> lr) & 1)) put(dk, a.scale, dko, pk);
    if (key < a.S && !((againv >> lr) & 1)) put(dv, 1.f, dvo, pv);
    // Keys again, over this block's steps: lanes are queries for P and dS and dims for the sums.
    for (uint32_t again = againk | againv; again; again &= again - 1) {
        const int bit = __builtin_ctz(again), ra = 32 * kw + bit, rk = n0 + ra;
        const bool wantk = (againk >> bit) & 1, wantv = (againv >> bit) & 1;
        const T *k1 = kb + rk * a.ks[2], *v1 = vb + rk * a.vs[2];
        // A NaN lse of a query that sees the key is in P, it and a NaN dsum in dS: the key's sums are NaN.
        bool lostk = !wantk, lostv = !wantv;
        for (int i = i0; i < i1 && !(lostk && lostv); ++i) {
            const int h = hk * a.repeat + i / per_head, l = l0 + i % per_head * QM + lane;
            const bool ok = lane < QM && l < a.L && sees(a.offset + l, rk, a.window, a.sinks);
            const int64_t row = ((int64_t)b * a.H + h) * a.L + l;
            const float lse = ok ? a.lse_in[row] : 0.f, rs = ok ? a.dsum[row] : 0.f;
            lostv |= (bool)__any(lse != lse), lostk |= (bool)__any(lse != lse || rs != rs);
        }
        float xk[2], xv[2];
        xk[0] = xk[1] = lostk ? NAN : 0.f, xv[0] = xv[1] = lostv ? NAN : 0.f;
        for (int i = i0; i < i1 && !(all_nan(lane, a.E, xk[0], xk[1]) && all_nan(lane, a.E, xv[0], xv[1])); ++i) {
            const int h = hk * a.repeat + i / per_head, m = l0 + i % per_head * QM, l = m + lane;
            const bool ok = lane < QM && l < a.L && sees(a.offset + l, rk, a.window, a.sinks);
            float pr = 0.f, ds = 0.f;
            if (ok) {
                const int64_t row = ((int64_t)b * a.H + h) * a.L + l;
                pr = exp2_fast((plain_dot<T>(qb + h * a.qs[1] + l * a.qs[2], k1, a.E) * a.scale - a.lse_in[row]) * kLog2e);
                ds = pr * (plain_dot<T>(gb + h * a.gs[1] + l * a.gs[2], v1, a.E) - a.dsum[row]);
            }
            for (uint64_t left = __ballot(ok); left; left &= left - 1) {
                const int j = __builtin_ctzll(left);
                const float pj = __shfl(pr, j, 64), dj = __shfl(ds, j, 64);
                const T *q1 = qb + h * a.qs[1] + (m + j) * a.qs[2], *g1 = gb + h * a.gs[1] + (m + j) * a.gs[2];
#pragma unroll
                for (int d = lane, n = 0; n < 2; ++n, d += 64)
                    if (d < a.E) xk[n] = fmaf(dj, to_f32<T>(q1[d]), xk[n]), xv[n] = fmaf(pj, to_f32<T>(g1[d]), xv[n]);
            }
        }
#pragma unroll
        for (int d = lane, n = 0; n < 2; ++n, d += 64) {
            if (d >= a.E) continue;
            if (wantk) {
                if (pcs.n > 1) pk[ra * a.E + d] = xk[n] * a.scale;
                else dko[(int64_t)ra * a.E + d] = from_f32<T>(xk[n] * a.scale);
            }
            if (wantv) {
                if (pcs.n > 1) pv[ra * a.E + d] = xv[n];
                else dvo[(int64_t)ra * a.E + d] = from_f32<T>(xv[n]);
            }
        }
    }
}

// The pieces of each key row summed in order, one thread per 4 dims of a row of dK or dV: the first `rows`
// keys of every kv head.
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WinArgs a, int rows) {
    const int groups = (a.E + 3) / 4, nkt = (a.S + kM - 1) / kM;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.B * a.Hkv * rows * groups * 2;
    if (id >= n) return;
    const int d = (int)(id % groups) * 4, which = (int)(id / groups % 2);
    const int64_t r = id / groups / 2;
    const int key = (int)(r % rows), bhk = (int)(r / rows);
    const Pieces pcs = pieces_of(a, nkt, bhk, key / kM);
    const float *src = a.kv_part + (pcs.slot * 2 + which) * kM * a.E + (int64_t)(key % kM) * a.E + d;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < pcs.n; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.E) x[e] += src[(int64_t)i * 2 * kM * a.E + e];
    T *dst = static_cast<T *>(which ? a.dv : a.dk) + ((int64_t)bhk * a.S + key) * a.E;
    store4<T, false>(dst, d, a.E, x[0], x[1], x[2], x[3]);
}

// How the dK / dV grid is cut.  A tile of sinks has the queries of the whole sequence where the others have a
// window's: pieces of about as many steps as those.  And where the blocks do not fill the CUs, pieces
// of at least 4 steps that do.  bf16 E128: a step of B2 H32/8 L8192 W1024 with 4 sinks took 6.5 ms with a sink
// tile's queries in one workgroup and 2.5 in pieces; the gradient of B1 H8/2 L1024 W256 90 us without pieces or with
// pieces of 16 steps, 56 with those of 4.
void plan_pieces(WinArgs &a, bool bf16) {
    const int QM = bf16 || a.E <= 64 ? 64 : 32, nkt = (a.S + kM - 1) / kM;
    a.sink_tiles = (int)std::min<int64_t>(nkt, ((int64_t)a.sinks + kM - 1) / kM);
    a.sink_pieces = a.tile_pieces = 1;
    if (nkt == 0 || a.L == 0 || a.B * a.Hkv == 0) return;
    // Steps of the longest tile without sinks: its queries grow in number up to the tile of the first query's
    // position, and do not behind the next.
    int64_t most = 0;
    for (int kt = a.offset / kM; kt <= a.offset / kM + 1 && nkt > a.sink_tiles; ++kt)
        most = std::max(most, tile_steps(a, std::clamp(kt, a.sink_tiles, nkt - 1) * kM, QM));
    const int64_t heads = (int64_t)a.B * a.Hkv, cus = std::max(device_cus(), 1), rest = nkt - a.sink_tiles;
    if (rest > 0 && most > 0)
        a.tile_pieces = (int)std::max<int64_t>(1, std::min<int64_t>(most / 4, cus / (heads * rest)));
    const int64_t sink = a.sink_tiles > 0 ? tile_steps(a, 0, QM) : 0;
    const int64_t piece = std::max<int64_t>(4, rest > 0 && most > 0 ? (most + a.tile_pieces - 1) / a.tile_pieces : sink);
    if (rest == 0 && sink > 0) {
        a.sink_pieces = (int)std::max<int64_t>(1, std::min<int64_t>(sink / 4, cus / (heads * a.sink_tiles)));
    } else if (sink > 0) {  // (no more than 4 blocks per CU: the partials stay below 140 MB)
        const int64_t room = 4 * cus / (heads * a.sink_tiles);
        a.sink_pieces = (int)std::max<int64_t>(1, std::min<int64_t>(room, (sink + piece - 1) / piece));
    }
}

int64_t blocks_per_head(const WinArgs &a) {
    const int nkt = (a.S + kM - 1) / kM;
    return (int64_t)a.sink_tiles * a.sink_pieces + (int64_t)(nkt - a.sink_tiles) * a.tile_pieces;
}

template <typename T, int D, bool VEC>
hipError_t launch_v(const WinArgs &a, hipStream_t st) {
    if (a.L > 0)
        return_if(launch(window_dq_kernel<T, D, VEC>, dim3((unsigned)((int64_t)(a.L + kM - 1) / kM * a.B * a.H)), dim3(kThreads),
                         st, a));
    if (a.S == 0) return hipSuccess;
    return_if(launch(window_dkdv_kernel<T, D, VEC>, dim3((unsigned)(blocks_per_head(a) * a.B * a.Hkv)),
                     dim3(kThreads * kHalves<T, D>), st, a));
    const int rows = a.tile_pieces > 1 ? a.S : a.sink_pieces > 1 ? std::min(a.S, a.sink_tiles * kM) : 0;
    if (rows == 0) return hipSuccess;
    const int64_t n = (int64_t)a.B * a.Hkv * rows * ((a.E + 3) / 4) * 2;
    return launch(window_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), st, a, rows);
}
template <typename T, int D>
hipError_t launch_d(const WinArgs &a, hipStream_t st) {
    return a.vec ? launch_v<T, D, true>(a, st) : launch_v<T, D, false>(a, st);
}
template <typename T>
hipError_t launch_t(const WinArgs &a, hipStream_t st) {
    if (a.E <= 32) return launch_d<T, 32>(a, st);
    if (a.E <= 64) return launch_d<T, 64>(a, st);
    return launch_d<T, 128>(a, st);
}

}  // namespace

size_t window_bwd_part_bytes(const WinArgs &args, bool bf16) {
    WinArgs a = args;
    plan_pieces(a, bf16);
    if (a.sink_pieces == 1 && a.tile_pieces == 1) return 0;
    return (size_t)(blocks_per_head(a) * a.B * a.Hkv) * 2 * kM * a.E * sizeof(float);
}

hipError_t launch_window_bwd(const WinArgs &args, bool bf16, hipStream_t st) {
    WinArgs a = args;
    plan_pieces(a, bf16);
    return bf16 ? launch_t<__bf16>(a, st) : launch_t<float>(a, st);
}

}  // namespace dc
