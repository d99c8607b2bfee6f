// One query per sequence over a KV cache with a window and sinks (dc_window_decode): bound by reading the
// visible rows of K and V once.
//
// A cache row belongs to LPR lanes, each with one 16-byte piece; a wave reads 64 / LPR rows at a time, U
// times over, K and V together.  The REP query heads of a workgroup share those registers.  A group of
// lanes keeps a softmax state of its own (maximum, sum, its dims of the output) over the keys it meets;
// groups, waves and the pieces that a sequence's keys are split into are joined at the end.
// Rows behind a sequence's length or outside the window are never read.
//
// Probabilities are formed as 2^(score - maximum - 16), so that up to 65536 of them times values near the
// type's largest do not overflow before the division by their sum.
#include <algorithm>

#include "params.hpp"
#include "window.hpp"

namespace dc {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kUnroll = 4;
constexpr float kShift = 16.f;

template <typename T, int CH, bool VEC>
DEVI void load_piece(const T *row, int d0, int E, float (&x)[CH]) {
    if constexpr (VEC) {
        typedef T vec __attribute__((ext_vector_type(CH)));
        if (d0 >= E) {
#pragma unroll
            for (int e = 0; e < CH; ++e) x[e] = 0.f;
            return;
        }
        const vec r = *reinterpret_cast<const vec *>(row + d0);
#pragma unroll
        for (int e = 0; e < CH; ++e) x[e] = to_f32<T>(r[e]);
    } else {
#pragma unroll
        for (int e = 0; e < CH; ++e) x[e] = d0 + e < E ? to_f32<T>(row[d0 + e]) : 0.f;
    }
}

// The keys the query of sequence b sees: ns sinks, then those from lo on; n in all.
struct Seen {
    int ns, lo, n;
    DEVI int key(int j) const { return j < ns ? j : lo + (j - ns); }
};
DEVI Seen seen_by(const WinDecodeArgs &a, int b) {
    int64_t len = a.S;
    if (a.length_bytes == 4) len = static_cast<const int32_t *>(a.lengths)[b];
    else if (a.length_bytes == 8) len = static_cast<const int64_t *>(a.lengths)[b];
    const int n = (int)(len < 0 ? 0 : len > a.S ? a.S : len);
    Seen s;
    s.lo = n > a.window ? n - a.window : 0;
    s.ns = min(a.sinks, s.lo);
    s.n = s.ns + (n - s.lo);
    return s;
}

template <typename T, int LPR, int REP, bool VEC>
__global__ __launch_bounds__(kThreads) void window_decode_kernel(WinDecodeArgs a) {
    constexpr int CH = 16 / sizeof(T), GW = 64 / LPR, STEP = kWaves * GW, U = kUnroll;
    __shared__ float sm[kWaves][REP], ssum[kWaves][REP], so[kWaves][REP][LPR * CH];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = lane % LPR, grp = lane / LPR;
    const int nhb = (a.repeat + REP - 1) / REP;
    int w = blockIdx.x;
    const int piece = w % a.splits;
    w /= a.splits;
    const int hb = w % nhb;
    w /= nhb;
    const int hk = w % a.Hkv, b = w / a.Hkv;
    const int h0 = hk * a.repeat + hb * REP, nh = min(REP, a.repeat - hb * REP);
    const Seen seen = seen_by(a, b);
    const int j0 = (int)((int64_t)piece * seen.n / a.splits), j1 = (int)((int64_t)(piece + 1) * seen.n / a.splits);
    const T *kb = static_cast<const T *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T *vb = static_cast<const T *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const int d0 = sub * CH;

    float q[REP][CH], acc[REP][CH], m[REP], sum[REP];
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        load_piece<T, CH, VEC>(static_cast<const T *>(a.q) + b * a.qs[0] + (h0 + min(r, nh - 1)) * a.qs[1], d0, a.E, q[r]);
        m[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
        for (int e = 0; e < CH; ++e) q[r][e] *= a.scale_log2, acc[r][e] = 0.f;
    }
    for (int base = j0 + wave * GW + grp; base - (wave * GW + grp) < j1; base += U * STEP) {
        float k[U][CH], v[U][CH];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = seen.key(min(base + u * STEP, j1 - 1));
            load_piece<T, CH, VEC>(kb + key * a.ks[2], d0, a.E, k[u]);
            load_piece<T, CH, VEC>(vb + key * a.vs[2], d0, a.E, v[u]);
        }
#pragma unroll
        for (int r = 0; r < REP; ++r) {
            float s[U], top = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < CH; ++e) x = fmaf(q[r][e], k[u][e], x);
                s[u] = base + u * STEP < j1 ? lanes_sum<LPR>(x) : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            // (alpha: m's own 2^-16 is in sum and acc already.)
            const float ref = top == -INFINITY ? 0.f : top, alpha = exp2_fast(m[r] - ref);
            m[r] = top, sum[r] *= alpha;
#pragma unroll
            for (int e = 0; e < CH; ++e) acc[r][e] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // (A key past the end repeats a visible one, with nothing of it.)
                const float p = base + u * STEP < j1 ? exp2_fast(s[u] - ref - kShift) : 0.f;
                sum[r] += p;
#pragma unroll
                for (int e = 0; e < CH; ++e) acc[r][e] = fmaf(p, v[u][e], acc[r][e]);
            }
        }
    }
    // The groups of the wave.
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        float top = m[r];
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float f = exp2_fast(m[r] - (top == -INFINITY ? 0.f : top));
        float t = sum[r] * f;
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            float x = acc[r][e] * f;
#pragma unroll
            for (int o = LPR; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
            if (grp == 0) so[wave][r][d0 + e] = x;
        }
        if (lane == 0) sm[wave][r] = top, ssum[wave][r] = t;
    }
    __syncthreads();
    // The waves; then the result, or this piece's share of it: output, maximum, sum.
    for (int i = tid; i < nh * LPR * CH; i += kThreads) {
        const int r = i / (LPR * CH), d = i % (LPR * CH);
        float top = sm[0][r];
#pragma unroll
        for (int x = 1; x < kWaves; ++x) top = fmaxf(top, sm[x][r]);
        const float ref = top == -INFINITY ? 0.f : top;
        float o = 0.f, t = 0.f;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            const float f = exp2_fast(sm[x][r] - ref);
            o = fmaf(f, so[x][r][d], o), t = fmaf(f, ssum[x][r], t);
        }
        const int64_t row = (int64_t)b * a.H + h0 + r;
        if (a.splits > 1) {
            float *part = a.part + (row * a.splits + piece) * (a.E + 2);
            if (d < a.E) part[d] = o;
            if (d == 0) part[a.E] = top, part[a.E + 1] = t;
        } else {
            if (d < a.E) static_cast<T *>(a.out)[row * a.E + d] = from_f32<T>(t == 0.f ? 0.f : o / t);
            if (d == 0) a.lse[row] = t == 0.f ? 0.f : (ref + kShift + log2_fast(t)) * kLn2;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(64) void window_decode_merge_kernel(WinDecodeArgs a) {
    const int64_t row = blockIdx.x;
    const float *part = a.part + row * a.splits * (a.E + 2);
    float top = -INFINITY, t = 0.f;
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, part[i * (a.E + 2) + a.E]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int i = 0; i < a.splits; ++i) t = fmaf(exp2_fast(part[i * (a.E + 2) + a.E] - ref), part[i * (a.E + 2) + a.E + 1], t);
    for (int d = threadIdx.x; d < a.E; d += 64) {
        float o = 0.f;
        for (int i = 0; i < a.splits; ++i) o = fmaf(exp2_fast(part[i * (a.E + 2) + a.E] - ref), part[i * (a.E + 2) + d], o);
        static_cast<T *>(a.out)[row * a.E + d] = from_f32<T>(t == 0.f ? 0.f : o / t);
    }
    if (threadIdx.x == 0) a.lse[row] = t == 0.f ? 0.f : (ref + kShift + log2_fast(t)) * kLn2;
}

int heads_per_block(int repeat) { return repeat >= 5 ? 8 : repeat >= 3 ? 4 : repeat; }

template <typename T, int LPR, int REP, bool VEC>
hipError_t launch_r(const WinDecodeArgs &a, hipStream_t st) {
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.repeat + REP - 1) / REP) * a.splits;
    return_if(launch(window_decode_kernel<T, LPR, REP, VEC>, dim3((unsigned)blocks), dim3(kThreads), st, a));
    if (a.splits == 1) return hipSuccess;
    return launch(window_decode_merge_kernel<T>, dim3((unsigned)((int64_t)a.B * a.H)), dim3(64), st, a);
}
template <typename T, int LPR, bool VEC>
hipError_t launch_l(const WinDecodeArgs &a, hipStream_t st) {
    switch (heads_per_block(a.repeat)) {
        case 1: return launch_r<T, LPR, 1, VEC>(a, st);
        case 2: return launch_r<T, LPR, 2, VEC>(a, st);
        case 4: return launch_r<T, LPR, 4, VEC>(a, st);
        default: return launch_r<T, LPR, 8, VEC>(a, st);
    }
}
template <typename T, bool VEC>
hipError_t launch_v(const WinDecodeArgs &a, hipStream_t st) {
    constexpr int CH = 16 / sizeof(T);
    if (a.E <= 8 * CH) return launch_l<T, 8, VEC>(a, st);
    if (a.E <= 16 * CH) return launch_l<T, 16, VEC>(a, st);
    if (a.E <= 32 * CH) return launch_l<T, 32, VEC>(a, st);
    if constexpr (CH == 4) return launch_l<T, 64, VEC>(a, st);
    return hipErrorInvalidValue;  // not reached: head dims up to 256
}

}  // namespace

// Pieces of a sequence's keys: as many as give every CU two workgroups, of at least 128 keys.
int window_decode_splits(const WinDecodeArgs &a, bool) {
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.repeat + heads_per_block(a.repeat) - 1) / heads_per_block(a.repeat));
    const int64_t span = std::min<int64_t>(a.S, (int64_t)a.window + a.sinks), cus = std::max(device_cus(), 1);
    if (blocks == 0) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>((span + 127) / 128, 2 * cus / blocks));
}

hipError_t launch_window_decode(const WinDecodeArgs &a, bool bf16, hipStream_t st) {
    if (bf16) return a.vec ? launch_v<__bf16, true>(a, st) : launch_v<__bf16, false>(a, st);
    return a.vec ? launch_v<float, true>(a, st) : launch_v<float, false>(a, st);
}

}  // namespace dc
