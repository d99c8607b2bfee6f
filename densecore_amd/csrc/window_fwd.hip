// Forward of attention with a sliding window and sinks (window.hpp): out = softmax over the visible
// keys of scale q k^T, times v, in one pass with a running maximum and sum.
//
// A workgroup of 4 waves owns 128 rows (queries) and visits only the key tiles one of them sees
// (Band): its window's and the sinks'.  A wave owns 32 rows, held in registers as the second operand of
// S^T = K Q^T, so a lane holds one row's softmax state; P goes straight from S^T's accumulators into
// O^T += V^T P^T.  K and V tiles are double-buffered in LDS.  Rows of short queries (a few tokens of
// each head that shares a kv head) are packed into one tile.
//
// Bound: a wave's own chain of transfers, products and softmax, two waves to a SIMD.  B2 H32/8 L8192 E128 W1024 bf16:
// 440 us, and 515 with the rest written, 500 TFLOP/s of the visible pairs' 4 E and 750 with P's lo terms (a library
// product of 8192^3 reaches 1139); MFMA busy 38%.  At a step that took 488 us, leaving out the maximum gave 474,
// the exponentials 425, P V 357, the transfers 385: no single one of them is what a wave waits for.  Float32 (six bf16
// products each) B8 H12 L1024 E64 W256: 76 us.
//
// Where a result is not finite (an infinite or NaN operand, which matrix products spread to rows
// that do not see it) the row is computed again in plain float32 over its visible keys alone.
#include <algorithm>

#include "params.hpp"
#include "window.hpp"

namespace dc {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kM = 32 * kWaves;
template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // keys per tile
template <typename T, int D>
constexpr int kWavesPerSimd = sizeof(T) == 2 || D <= 64 ? 2 : 1;  // LDS: 110 KB of float32 tiles at D = 128
// ... as the least.  bf16 at D = 64 runs four, whose products cover each other's softmax (B4 H32 L4096 W1024
// 262 -> 227 us against two), at D = 32 too (225 -> 165); at D = 128 two workgroups' tiles fill the LDS.

// Row r of a group of `pack`ed heads (or of one head) as (head within the group, query).
struct RowAt {
    int h, l;
};
DEVI RowAt row_at(const WinArgs &a, int r) { return a.pack ? RowAt{r / a.L, r % a.L} : RowAt{0, r}; }
// The first and last position of rows r0 .. r1.
DEVI void positions(const WinArgs &a, int r0, int r1, int &p0, int &p1) {
    if (a.pack && r0 / a.L != r1 / a.L) {
        p0 = a.offset, p1 = a.offset + a.L - 1;
    } else {
        p0 = a.offset + row_at(a, r0).l, p1 = a.offset + row_at(a, r1).l;
    }
}

// Element i of the result.
template <typename T>
DEVI void put(const WinArgs &a, int64_t i, float x) {
    static_cast<T *>(a.out)[i] = from_f32<T>(x);
    if (sizeof(T) == 2 && a.rest) static_cast<T *>(a.rest)[i] = from_f32<T>(rest_of(x));
}

// One row again, keys of tiles [i0, i1): lanes are keys for the scores and dims for the output
// (dims lane and lane + 64).  The maximum and sum first, so that the output is a sum of P / sum times v and
// does not overflow where the result does not.
template <typename T>
DEVI void plain_row(const WinArgs &a, const T *q, const T *kb, const T *vb, int p, Band band, int i0, int i1, int lane,
                    float (&o)[2], float &m, float &sum) {
    constexpr int BN = kKeys<T>;
    auto score = [&](int n0, bool &ok) {
        const int key = n0 + lane;
        ok = lane < BN && key < a.S && sees(p, key, a.window, a.sinks);
        return ok ? plain_dot<T>(q, kb + key * a.ks[2], a.E) * a.scale_log2 : -INFINITY;
    };
    o[0] = o[1] = sum = 0.f, m = -INFINITY;
    bool ok;
    for (int i = i0; i < i1; ++i) {
        const float s = score(band.tile(i) * BN, ok);
        const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.f : top;
        sum = sum * exp2_fast(m - base) + wave_sum(ok ? exp2_fast(s - base) : 0.f);
        m = top;
        if (sum != sum) {  // a score that is seen is NaN: so is the row, whatever follows
            o[0] = o[1] = sum;
            return;
        }
    }
    const float base = m == -INFINITY ? 0.f : m, inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int i = i0; i < i1; ++i) {
        const int n0 = band.tile(i) * BN;
        const float s = score(n0, ok), pr = ok ? exp2_fast(s - base) * inv : 0.f;
        for (uint64_t left = __ballot(ok); left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const float pj = __shfl(pr, j, 64);
            const T *v = vb + (n0 + j) * a.vs[2];
            if (lane < a.E) o[0] = fmaf(pj, to_f32<T>(v[lane]), o[0]);
            if (lane + 64 < a.E) o[1] = fmaf(pj, to_f32<T>(v[lane + 64]), o[1]);
        }
        if (all_nan(lane, a.E, o[0], o[1])) return;
    }
}

// The end of a wave: O / sum and lse of its 32 rows (from row wr0 of the group on, this lane's `row` of out),
// or the piece's share of them; rows that are not finite again.
template <typename T, int D, bool VEC>
DEVI void write_rows(const WinArgs &a, const f32x16 (&acc)[D / 32], float m_run, float l_part, int lane, int wr0, bool in,
                     int64_t row, int b, int h0, const T *kb, const T *vb, Band band, int i0, int i1, int piece, void *room) {
    constexpr int NDT = D / 32;
    const int lr = lane & 31, g = lane >> 5;
    const float l_run = xor32_add(l_part);
    const bool empty = l_run == 0.f;
    const float inv = empty ? 0.f : 1.f / l_run;
    float test = l_run * 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) test += not_finite(acc[dt]);
    const uint64_t wrong = __ballot(in && test != 0.f);
    uint32_t again = (uint32_t)wrong | (uint32_t)(wrong >> 32);
    const int64_t nrows = (int64_t)a.B * a.H * a.L;
    if constexpr (kTurned<T, D, VEC>) {
        if (a.splits == 1) {
            const int rows = (a.pack ? a.repeat : 1) * a.L;
            auto to = [&](void *base) {
                return [&, base](int r) -> __bf16 * {
                    if (wr0 + r >= rows || ((again >> r) & 1)) return nullptr;
                    const RowAt ra = row_at(a, wr0 + r);
                    return static_cast<__bf16 *>(base) + (((int64_t)b * a.H + h0 + ra.h) * a.L + ra.l) * a.E;
                };
            };
            u32x4 *const turn = static_cast<u32x4 *>(room);
            store_turned<D>(turn, lane, a.E, [&](int dt, int e) { return acc[dt][e] * inv; }, to(a.out));
            if (a.rest) store_turned<D>(turn, lane, a.E, [&](int dt, int e) { return rest_of(acc[dt][e] * inv); }, to(a.rest));
        }
    }
    if (in && !((again >> lr) & 1)) {
        const float lse = (m_run + log2_fast(l_run)) * kLn2;
        if (a.splits > 1) {
            const int64_t slot = piece * nrows + row;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    store4<float, VEC>(a.part + slot * a.E, dt * 32 + acc_row(e, g), a.E, acc[dt][e] * inv, acc[dt][e + 1] * inv,
                                       acc[dt][e + 2] * inv, acc[dt][e + 3] * inv);
            if (g == 0) a.part_lse[slot] = empty ? -INFINITY : lse;
        } else {
            if constexpr (!kTurned<T, D, VEC>) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int d = dt * 32 + acc_row(e, g);
                    const float x0 = acc[dt][e] * inv, x1 = acc[dt][e + 1] * inv, x2 = acc[dt][e + 2] * inv,
                                x3 = acc[dt][e + 3] * inv;
                    store4<T, VEC>(static_cast<T *>(a.out) + row * a.E, d, a.E, x0, x1, x2, x3);
                    if (sizeof(T) == 2 && a.rest)
                        store4<T, VEC>(static_cast<T *>(a.rest) + row * a.E, d, a.E, rest_of(x0), rest_of(x1), rest_of(x2),
                                       rest_of(x3));
                }
            }
            if (g == 0) a.lse[row] = empty ? 0.f : lse;
        }
    }
    for (; again; again &= again - 1) {
        const int rr = wr0 + __builtin_ctz(again);
        const RowAt ra = row_at(a, rr);
        const int64_t orow = ((int64_t)b * a.H + h0 + ra.h) * a.L + ra.l;
        float o[2], m, sum;
        plain_row<T>(a, static_cast<const T *>(a.q) + b * a.qs[0] + (h0 + ra.h) * a.qs[1] + ra.l * a.qs[2], kb, vb,
                     a.offset + ra.l, band, i0, i1, lane, o, m, sum);
        const bool none = sum == 0.f;
        const float lse = (m + log2_fast(sum)) * kLn2;
        const int64_t slot = piece * nrows + orow;
#pragma unroll
        for (int d = lane, j = 0; j < 2; ++j, d += 64) {
            if (d >= a.E) continue;
            if (a.splits > 1) a.part[slot * a.E + d] = o[j];
            else put<T>(a, orow * a.E + d, o[j]);
        }
        if (lane == 0) {
            if (a.splits > 1) a.part_lse[slot] = none ? -INFINITY : lse;
            else a.lse[orow] = none ? 0.f : lse;
        }
    }
}

template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, D>))) void window_fwd_kernel(WinArgs a) {
    typedef Ops<T> O;
    constexpr int BN = kKeys<T>, NT = BN / 32, KSTEP = D / 16, NDT = D / 32;
    typedef Stage<T, BN, D, kThreads, VEC> St;
    __shared__ typename St::Tile sk[2], sv[2];
    static_assert(!kTurned<T, D, VEC> || sizeof(sk) >= kWaves * kRoom<D> * sizeof(u32x4), "the results' turn");

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.pack ? a.repeat : 1, rows = G * a.L;
    const int nqt = (rows + kM - 1) / kM;
    int w = logical_block();
    const int piece = w % a.splits;
    w /= a.splits;
    // The heads (groups of heads) of a kv head side by side, then its row tiles, longest first: the workgroups
    // an XCD runs at once read few keys.
    const int share = a.repeat / G;
    const int qt = nqt - 1 - w / share % nqt, kvh = w / share / nqt;
    const int b = kvh / a.Hkv, hk = kvh % a.Hkv, h0 = hk * a.repeat + w % share * G;
    const int r0 = qt * kM, wr0 = r0 + 32 * wave, r = wr0 + lr;
    const bool in = r < rows;
    const RowAt at = row_at(a, in ? r : rows - 1);
    const int p = in ? a.offset + at.l : -1;  // -1: sees nothing
    const int64_t row = ((int64_t)b * a.H + h0 + at.h) * a.L + at.l;  // of out and lse

    int p0, p1, wp0 = 0, wp1 = -1;  // positions of the workgroup's rows and of the wave's (none: empty)
    positions(a, r0, min(r0 + kM, rows) - 1, p0, p1);
    if (wr0 < rows) positions(a, wr0, min(wr0 + 32, rows) - 1, wp0, wp1);
    const Band band = band_of(p0, p1, a.S, a.window, a.sinks, BN);
    const int i0 = (int)((int64_t)piece * band.n / a.splits), i1 = (int)((int64_t)(piece + 1) * band.n / a.splits);

    const T *kb = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T *vb = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + (h0 + at.h) * a.qs[1] + at.l * a.qs[2];

    const uint32_t rowb = row_lanebase<BN, D>(lane), trb = tr_lanebase<BN, D>(lane);
    St kst, vst;
    auto start = [&](int i) {
        const int n0 = band.tile(i) * BN, nr = min(BN, a.S - n0), buf = (i - i0) & 1;
        kst.start(sk[buf], kb + (int64_t)n0 * a.ks[2], a.ks[2], nr, a.E, tid);
        vst.start(sv[buf], vb + (int64_t)n0 * a.vs[2], a.vs[2], nr, a.E, tid);
    };
    auto finish = [&](int i) {
        kst.finish(sk[(i - i0) & 1], tid);
        vst.finish(sv[(i - i0) & 1], tid);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) St::clear(sk[i], a.E, tid), St::clear(sv[i], a.E, tid);
    if (i0 < i1) start(i0);  // on its way while the queries load

    // Scores are fma(q.k, c, -m) in base 2; a negative scale is a sign flip of the queries, and a zero
    // one the smallest normal number (every visible key then gets P = 1).
    const float c = fmaxf(fabsf(a.scale_log2), 0x1p-126f);
    typename O::Frag qf[KSTEP];
#pragma unroll
    for (int t = 0; t < KSTEP; ++t) {
        qf[t] = O::template load<VEC>(q, 16 * t + 8 * g, a.E, in);
        if (a.scale_log2 < 0.f) qf[t] = O::neg(qf[t]);
    }
    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
    float m_run = -INFINITY, l_part = 0.f;  // l_part: this half-wave's keys only

    if (i0 < i1) finish(i0);

    auto step = [&](int i) {
        const int n0 = band.tile(i) * BN, buf = (i - i0) & 1;
        bool live[NT], any = false;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            const int k0 = n0 + 32 * kt;
            live[kt] = k0 < a.S && k0 <= wp1 && (wp0 - (k0 + 31) < a.window || k0 < a.sinks);
            any |= live[kt];
        }
        if (!any) return;
        f32x16 s[NT];
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kt][e] = 0.f;
        }
        if (live[0] && live[NT - 1]) {
#pragma unroll
            for (int st = 0; st < KSTEP; ++st)
#pragma unroll
                for (int kt = 0; kt < NT; ++kt) s[kt] = O::mma(O::row(sk[buf], rowb, 32 * kt, st), qf[st], s[kt]);
            reads_ahead<KSTEP * NT, O::MMAS, O::READS, sizeof(T) == 2 ? 4 : 2>();
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) pin(s[kt]);
            __builtin_amdgcn_sched_barrier(0);
        } else {
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) {
                if (!live[kt]) continue;
#pragma unroll
                for (int st = 0; st < KSTEP; ++st) s[kt] = O::mma(O::row(sk[buf], rowb, 32 * kt, st), qf[st], s[kt]);
            }
        }
        const bool all = n0 + BN <= a.S && n0 + BN - 1 <= wp0 && (wp1 - n0 < a.window || n0 + BN <= a.sinks);
        if (!all) {
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) {
                // (A sub-tile that is not live holds no product: all of it is hidden.)
                const SeenKeys seen(p, n0 + 32 * kt + 4 * g, a.S, a.window, a.sinks);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kt][e] = seen(acc_const(e)) ? s[kt][e] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kt][e]);
        mx = xor32_max(mx) * c;
        // The reference of the exponents moves only when some row's maximum exceeds it by more than 8.
        if (__any(mx > m_run + 8.f)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = exp2_fast(m_run - (m_new == -INFINITY ? 0.f : m_new));
            l_part *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[dt][e] *= alpha;
            m_run = m_new;
        }
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kt][e] = exp2_fast(fmaf(s[kt][e], c, neg_m));
                l_part += s[kt][e];
            }
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            if (!live[kt]) continue;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                typename O::Frag vf[NDT];
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) vf[dt] = O::tr(sv[buf], trb, 32 * kt + 16 * u, dt);
                O::mma_p(vf, s[kt], 8 * u, acc);
            }
        }
    };
    for (int i = i0; i < i1; ++i) {
        __syncthreads();  // tile i is there, and everyone is done with tile i - 1
        if (i + 1 < i1) start(i + 1);
        step(i);
        if (i + 1 < i1) finish(i + 1);
    }

    if (kTurned<T, D, VEC>) __syncthreads();  // everyone is done with the tiles, which the results now pass through
    write_rows<T, D, VEC>(a, acc, m_run, l_part, lane, wr0, in, row, b, h0, kb, vb, band, i0, i1, piece,
                          reinterpret_cast<u32x4 *>(sk) + wave * kRoom<D>);
}

// Joins the pieces of each row, 16 lanes per row: lse = log sum exp(lse_i), out = sum exp(lse_i - lse) o_i.
// The lanes form the pieces' weights once (LDS), then each sums 4 dims at a time.
constexpr int kMaxSplits = 128;
template <typename T, bool VEC4>
__global__ __launch_bounds__(256) void window_merge_kernel(WinArgs a) {
    __shared__ float weight[16][kMaxSplits + 1];
    const int64_t nrows = (int64_t)a.B * a.H * a.L, row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (row >= nrows) return;  // (whole groups of lanes; a row's weights are its own lanes' alone)
    const int part = threadIdx.x & 15, r = threadIdx.x >> 4;
    float top = -INFINITY;
    for (int i = part; i < a.splits; i += 16) top = fmaxf(top, weight[r][i] = a.part_lse[i * nrows + row]);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int i = part; i < a.splits; i += 16) sum += weight[r][i] = exp2_fast((weight[r][i] - base) * kLog2e);
    sum = lanes_sum<16>(sum);
    const bool empty = sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    wait_lds();
    for (int d = 4 * part; d < a.E; d += 64) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < a.splits; ++i) {
            const float *p = a.part + (i * nrows + row) * a.E + d, w = weight[r][i] * inv;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            if constexpr (VEC4) {
                x = *reinterpret_cast<const f32x4 *>(p);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = d + e < a.E ? p[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w, x[e], o[e]);
        }
        store4<T, false>(static_cast<T *>(a.out) + row * a.E, d, a.E, o[0], o[1], o[2], o[3]);
        if (sizeof(T) == 2 && a.rest)
            store4<T, false>(static_cast<T *>(a.rest) + row * a.E, d, a.E, rest_of(o[0]), rest_of(o[1]), rest_of(o[2]), rest_of(o[3]));
    }
    if (part == 0) a.lse[row] = empty ? 0.f : base + log2_fast(sum) * kLn2;
}

// Heads that share a kv head share tiles where a head's queries fill at most half of one: B64 H32/8, 16 rows each over
// 1124 keys bf16 66 us, 171 apart; 48 rows, B16, 44 and 59; with 100 rows it no longer matters (68, 68).
bool packs(const WinArgs &a) { return a.repeat > 1 && a.L <= kM / 2; }

int64_t blocks_of(const WinArgs &a, bool pack) {
    const int64_t rows = (int64_t)(pack ? a.repeat : 1) * a.L;
    return (rows + kM - 1) / kM * a.B * (a.H / (pack ? a.repeat : 1));
}

// Pieces of each tile's keys where the tiles fill at most half of the CUs: as many as give each CU a workgroup with
// 256 keys (64 in float32, whose products take six times as long), or two with twice and four times that.  The
// partials of every piece are written and read again, so more of them cost more than they give: B2 H32/8, 64 rows
// over 4160 keys bf16 33 us with 8 pieces of 8 tiles, 37 with 16; B1 H32/8, 256 rows over 8192 keys 78 us with 4 and
// 73 with 8; float32 B1 H8/2 E128, 20 rows over 500 keys 23 us with pieces of 64 keys, 53 with 256.
int plan_splits(const WinArgs &a, bool bf16) {
    const int64_t blocks = blocks_of(a, packs(a)), cus = device_cus();
    if (blocks == 0 || cus <= 0 || 2 * blocks > cus) return 1;
    const int64_t span = std::min<int64_t>(a.S, (int64_t)a.window + a.sinks + std::min(a.L, kM));
    const int64_t one = std::min<int64_t>(span / (bf16 ? 256 : 64), cus / blocks);
    const int64_t two = std::min<int64_t>(span / (bf16 ? 512 : 256), 2 * cus / blocks);
    return (int)std::min<int64_t>(std::max<int64_t>({one, two, 1}), kMaxSplits);
}

template <typename T, int D, bool VEC>
hipError_t launch_v(const WinArgs &a, hipStream_t st) {
    return_if(launch(window_fwd_kernel<T, D, VEC>, dim3((unsigned)(blocks_of(a, a.pack) * a.splits)), dim3(kThreads), st, a));
    if (a.splits == 1) return hipSuccess;
    const int64_t nrows = (int64_t)a.B * a.H * a.L;
    const dim3 grid((unsigned)((nrows + 15) / 16)), block(256);
    return a.E % 4 == 0 ? launch(window_merge_kernel<T, true>, grid, block, st, a)
                        : launch(window_merge_kernel<T, false>, grid, block, st, a);
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

size_t window_fwd_part_bytes(const WinArgs &a, bool bf16) {
    const int n = plan_splits(a, bf16);
    return n > 1 ? (size_t)n * a.B * a.H * a.L * (a.E + 1) * sizeof(float) : 0;
}

hipError_t launch_window_fwd(const WinArgs &args, bool bf16, size_t part_bytes, hipStream_t st) {
    WinArgs a = args;
    a.pack = packs(a);
    a.splits = plan_splits(a, bf16);
    if (a.splits > 1 && (!a.part || part_bytes < window_fwd_part_bytes(a, bf16))) a.splits = 1;
    if (a.splits > 1) a.part_lse = a.part + (size_t)a.splits * a.B * a.H * a.L * a.E;
    return bf16 ? launch_t<__bf16>(a, st) : launch_t<float>(a, st);
}

}  // namespace dc
