// Backward of attention with a sliding window and sinks (window.hpp): with P = exp(scale q k^T - lse) at
// the visible pairs, dsum = rowsum(dO * O) and dS = P (dO v^T - dsum),
//     dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,
// dK and dV summed over the query heads that share a kv head.  Two kernels, no atomics:
//   * window_dq_kernel (queries stay, the forward's structure) also forms dsum;
//   * window_dkdv_kernel (keys stay): a workgroup of 4 waves owns 128 keys, 32 per wave with K and V in
//     registers, and walks the queries that see one of them, head after head.
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
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 64 : 32;  // dK / dV: queries per step
template <typename T, int D>
constexpr int kWavesPerSimd = D <= 64 && sizeof(T) == 2 ? 2 : 1;

template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D>, kWavesPerSimd<T, D>))) void window_dq_kernel(WinArgs a) {
    typedef Ops<T> O;
    constexpr int BN = kKeys<T>, NT = BN / 32, KSTEP = D / 16, NDT = D / 32;
    typedef Stage<T, BN, D, kThreads, VEC> St;
    __shared__ typename St::Tile sk[2], sv[2];

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nqt = (a.L + kM - 1) / kM;
    const int w = logical_block();
    const int qt = nqt - 1 - w % nqt, bh = w / nqt;
    const int b = bh / a.H, h = bh % a.H, hk = h / a.repeat;
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

    typename O::Frag qf[KSTEP], gf[KSTEP];
    float dsum = 0.f;
#pragma unroll
    for (int t = 0; t < KSTEP; ++t) {
        qf[t] = O::template load<VEC>(qb + l * a.qs[2], 16 * t + 8 * g, a.E, in);
        gf[t] = O::template load<VEC>(gb + l * a.gs[2], 16 * t + 8 * g, a.E, in);
        dsum += O::dot(gf[t], O::template load<VEC>(ob + (int64_t)l * a.E, 16 * t + 8 * g, a.E, in));
    }
    dsum = xor32_add(dsum);
    if (in && g == 0) a.dsum[row] = dsum;
    const float nlse = in ? -a.lse_in[row] * kLog2e : 0.f;

    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;

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
    if (band.n > 0) start(0), finish(0);

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
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = k0 + acc_row(e, g);
                float x = fmaf(s[e], a.scale_log2, nlse);
                const bool hidden = !all && (key >= a.S || !sees(p, key, a.window, a.sinks));
                s[e] = hidden ? 0.f : exp2_fast(x) * t[e];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename O::PFrag pf = O::split(s, 8 * u);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) acc[dt] = O::mma_p(O::tr(sk[i & 1], trb, 32 * kt + 16 * u, dt), pf, acc[dt]);
            }
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
    if (in && !((again >> lr) & 1)) {
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
        const float rs = plain_dot<T>(g1, ob + (int64_t)rl * a.E, a.E), rlse = a.lse_in[rr];
        if (lane == 0) a.dsum[rr] = rs;
        float o[2] = {0.f, 0.f};
        for (int i = 0; i < band.n; ++i) {
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

template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D>, kWavesPerSimd<T, D>))) void window_dkdv_kernel(WinArgs a) {
    typedef Ops<T> O;
    constexpr int QM = kRows<T>, NS = QM / 32, KSTEP = D / 16, NDT = D / 32;
    typedef Stage<T, QM, D, kThreads, VEC> St;
    __shared__ typename St::Tile sq[2], sg[2];
    __shared__ float slse[2][QM], sdsum[2][QM];  // -lse log2 e (-inf behind the last row: P = 0) and -dsum

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nkt = (a.S + kM - 1) / kM;
    const int w = logical_block();
    const int n0 = w % nkt * kM, bhk = w / nkt, b = bhk / a.Hkv, hk = bhk % a.Hkv;
    const int kw0 = n0 + 32 * wave, key = kw0 + lr;
    const T *kb = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T *vb = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const T *qb = static_cast<const T *>(a.q) + b * a.qs[0];
    const T *gb = static_cast<const T *>(a.dout) + b * a.gs[0];
    int l0, l1;
    query_range(a, n0, min(n0 + kM, a.S), l0, l1);
    const int per_head = (l1 - l0 + QM - 1) / QM, steps = per_head * a.repeat;

    St qst, gst;
    float stat = 0.f;
    auto start = [&](int i) {
        const int h = hk * a.repeat + i / per_head, m0 = l0 + i % per_head * QM, nr = min(QM, a.L - m0);
        qst.start(sq[i & 1], qb + h * a.qs[1] + m0 * a.qs[2], a.qs[2], nr, a.E, tid);
        gst.start(sg[i & 1], gb + h * a.gs[1] + m0 * a.gs[2], a.gs[2], nr, a.E, tid);
        if (tid < 2 * QM) {
            const int64_t row = ((int64_t)b * a.H + h) * a.L + m0 + tid % QM;
            if (tid < QM) stat = tid < nr ? -a.lse_in[row] * kLog2e : -INFINITY;
            else stat = tid - QM < nr ? -a.dsum[row] : 0.f;
        }
    };
    auto finish = [&](int i) {
        qst.finish(sq[i & 1], tid);
        gst.finish(sg[i & 1], tid);
        if (tid < QM) slse[i & 1][tid] = stat;
        else if (tid < 2 * QM) sdsum[i & 1][tid - QM] = stat;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) St::clear(sq[i], a.E, tid), St::clear(sg[i], a.E, tid);
    if (steps > 0) start(0), finish(0);

    typename O::Frag kf[KSTEP], vf[KSTEP];
#pragma unroll
    for (int t = 0; t < KSTEP; ++t) {
        const int kr = min(key, a.S - 1);
        kf[t] = O::template load<VEC>(kb + kr * a.ks[2], 16 * t + 8 * g, a.E, key < a.S);
        vf[t] = O::template load<VEC>(vb + kr * a.vs[2], 16 * t + 8 * g, a.E, key < a.S);
    }
    f32x16 dk[NDT], dv[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.f;
    const uint32_t rowb = row_lanebase<QM, D>(lane), trb = tr_lanebase<QM, D>(lane);

    auto step = [&](int i) {
        const int buf = i & 1, m0 = l0 + i % per_head * QM;
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
            const int mq = m0 + 32 * sub, q0 = a.offset + mq, q1 = a.offset + min(mq + 31, a.L - 1);
            if (mq >= a.L || kw0 >= a.S || kw0 > q1 || (q0 - (kw0 + 31) >= a.window && kw0 >= a.sinks)) continue;
            const bool all = kw0 + 31 < a.S && kw0 + 31 <= q0 && (q1 - kw0 < a.window || kw0 + 31 < a.sinks);
            f32x16 s, t;
            f32x4 nl[4];
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int rr = 32 * sub + 8 * r4 + 4 * g;
                const f32x4 nd = *reinterpret_cast<const f32x4 *>(&sdsum[buf][rr]);
                nl[r4] = *reinterpret_cast<const f32x4 *>(&slse[buf][rr]);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * r4 + j] = 0.f, t[4 * r4 + j] = nd[j];
            }
#pragma unroll
            for (int st = 0; st < KSTEP; ++st) {
                s = O::mma(O::row(sq[buf], rowb, 32 * sub, st), kf[st], s);
                t = O::mma(O::row(sg[buf], rowb, 32 * sub, st), vf[st], t);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int qp = q0 + acc_row(e, g);
                const bool hidden = !all && (key >= a.S || !sees(qp, key, a.window, a.sinks));
                const float pr = hidden ? 0.f : exp2_fast(fmaf(s[e], a.scale_log2, nl[e >> 2][e & 3]));
                s[e] = pr;
                t[e] = hidden ? 0.f : pr * t[e];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename O::PFrag pf = O::split(s, 8 * u), df = O::split(t, 8 * u);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) dv[dt] = O::mma_p(O::tr(sg[buf], trb, 32 * sub + 16 * u, dt), pf, dv[dt]);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) dk[dt] = O::mma_p(O::tr(sq[buf], trb, 32 * sub + 16 * u, dt), df, dk[dt]);
            }
        }
    };
    for (int i = 0; i < steps; ++i) {
        __syncthreads();
        if (i + 1 < steps) start(i + 1);
        step(i);
        if (i + 1 < steps) finish(i + 1);
    }

    float test = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) test += not_finite(dk[dt]) + not_finite(dv[dt]);
    const uint64_t wrong = __ballot(key < a.S && test != 0.f);
    uint32_t again = (uint32_t)wrong | (uint32_t)(wrong >> 32);
    T *dko = static_cast<T *>(a.dk) + (int64_t)bhk * a.S * a.E, *dvo = static_cast<T *>(a.dv) + (int64_t)bhk * a.S * a.E;
    if (key < a.S && !((again >> lr) & 1)) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = dt * 32 + acc_row(e, g);
                store4<T, VEC>(dko + (int64_t)key * a.E, d, a.E, dk[dt][e] * a.scale, dk[dt][e + 1] * a.scale,
                               dk[dt][e + 2] * a.scale, dk[dt][e + 3] * a.scale);
                store4<T, VEC>(dvo + (int64_t)key * a.E, d, a.E, dv[dt][e], dv[dt][e + 1], dv[dt][e + 2], dv[dt][e + 3]);
            }
    }
    // Keys again: lanes are queries for P and dS and dims for the sums.
    for (; again; again &= again - 1) {
        const int rk = kw0 + __builtin_ctz(again);
        const T *k1 = kb + rk * a.ks[2], *v1 = vb + rk * a.vs[2];
        float xk[2] = {0.f, 0.f}, xv[2] = {0.f, 0.f};
        for (int i = 0; i < a.repeat; ++i) {
            const int h = hk * a.repeat + i;
            for (int m = l0; m < l1; m += 64) {
                const int l = m + lane;
                const bool ok = l < l1 && sees(a.offset + l, rk, a.window, a.sinks);
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
        }
#pragma unroll
        for (int d = lane, n = 0; n < 2; ++n, d += 64)
            if (d < a.E) {
                dko[(int64_t)rk * a.E + d] = from_f32<T>(xk[n] * a.scale);
                dvo[(int64_t)rk * a.E + d] = from_f32<T>(xv[n]);
            }
    }
}

template <typename T, int D, bool VEC>
hipError_t launch_v(const WinArgs &a, hipStream_t st) {
    if (a.L > 0)
        return_if(launch(window_dq_kernel<T, D, VEC>, dim3((unsigned)((int64_t)(a.L + kM - 1) / kM * a.B * a.H)), dim3(kThreads),
                         st, a));
    if (a.S > 0)
        return_if(launch(window_dkdv_kernel<T, D, VEC>, dim3((unsigned)((int64_t)(a.S + kM - 1) / kM * a.B * a.Hkv)),
                         dim3(kThreads), st, a));
    return hipSuccess;
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

hipError_t launch_window_bwd(const WinArgs &a, bool bf16, hipStream_t st) {
    return bf16 ? launch_t<__bf16>(a, st) : launch_t<float>(a, st);
}

}  // namespace dc
