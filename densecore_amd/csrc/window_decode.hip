// One query per sequence over a KV cache with a window and sinks (dc_window_decode): bound by reading the
// visible rows of K and V once.  Float32 B8 H32/8 E128, 4096 keys: 51 us, 5.2 TB/s; bf16 B16: 57 us for a call, its two
// kernels 45 + 5 (269 MB, 6.0 TB/s in the first).
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

// A lane's piece of a row, as it lies: dims d0 .. d0 + CH - 1 (0 past E).
template <typename T, int CH, bool VEC>
struct Piece {
    typedef T vec __attribute__((ext_vector_type(CH)));
    vec x;
    DEVI void load(const T *row, int d0, int E) {
        if constexpr (VEC) {
            x = d0 < E ? *reinterpret_cast<const vec *>(row + d0) : vec(T(0));
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) x[e] = d0 + e < E ? row[d0 + e] : T(0);
        }
    }
    DEVI float operator[](int e) const { return to_f32<T>(x[e]); }
};

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

// Dim d of head r of a workgroup from its waves' ends (o: waves x heads x dims, m and sum: waves x heads): the
// result, or this piece's share of it: output, maximum, sum.
template <typename T>
DEVI void join_waves(const WinDecodeArgs &a, const float *o, const float *m, const float *sum, int heads, int dims, int b, int h0,
                     int piece, int r, int d) {
    float top = m[r];
#pragma unroll
    for (int x = 1; x < kWaves; ++x) top = fmaxf(top, m[x * heads + r]);
    const float ref = top == -INFINITY ? 0.f : top;
    float y = 0.f, t = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
        const float f = exp2_fast(m[x * heads + r] - ref);
        y = fmaf(f, o[(x * heads + r) * dims + d], y), t = fmaf(f, sum[x * heads + r], t);
    }
    const int64_t row = (int64_t)b * a.H + h0 + r;
    if (a.splits > 1) {
        float *part = a.part + (row * a.splits + piece) * (a.E + 2);
        if (d < a.E) part[d] = y;
        if (d == 0) part[a.E] = top, part[a.E + 1] = t;
    } else {
        if (d < a.E) static_cast<T *>(a.out)[row * a.E + d] = from_f32<T>(t == 0.f ? 0.f : y / t);
        if (d == 0) a.lse[row] = t == 0.f ? 0.f : (ref + kShift + log2_fast(t)) * kLn2;
    }
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
        Piece<T, CH, VEC> x;
        x.load(static_cast<const T *>(a.q) + b * a.qs[0] + (h0 + min(r, nh - 1)) * a.qs[1], d0, a.E);
        m[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
        for (int e = 0; e < CH; ++e) q[r][e] = x[e] * a.scale_log2, acc[r][e] = 0.f;
    }
    // The next keys' rows are on their way while these are computed.
    Piece<T, CH, VEC> k[U], v[U], k1[U], v1[U];
    auto load = [&](Piece<T, CH, VEC> (&kx)[U], Piece<T, CH, VEC> (&vx)[U], int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = base + u * STEP, key = seen.key(min(j, j1 - 1)), E = j < j1 ? a.E : 0;  // (past the end: zeros)
            kx[u].load(kb + key * a.ks[2], d0, E);
            vx[u].load(vb + key * a.vs[2], d0, E);
        }
    };
    const int mine = wave * GW + grp;
    if (j0 < j1) load(k, v, j0 + mine);
    for (int j = j0; j < j1; j += U * STEP) {
        const int base = j + mine;
        if (j + U * STEP < j1) load(k1, v1, base + U * STEP);
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
                const float p = base + u * STEP < j1 ? exp2_fast(s[u] - ref - kShift) : 0.f;
                sum[r] += p;
#pragma unroll
                for (int e = 0; e < CH; ++e) acc[r][e] = fmaf(p, v[u][e], acc[r][e]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = k1[u], v[u] = v1[u];
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
    for (int i = tid; i < nh * LPR * CH; i += kThreads)
        join_waves<T>(a, &so[0][0][0], &sm[0][0], &ssum[0][0], REP, LPR * CH, b, h0, piece, i / (LPR * CH), i % (LPR * CH));
}

// bf16 (16-byte pieces, head dims up to 128): the same, with the products on the matrix cores, so that the heads
// sharing a row (up to 16) cost next to nothing: 8 heads to a kv head are 150 VALU instructions for each 16 bytes
// of K and V in the kernel above, which is then bound by them (B8 H64/8 E128, 8192 keys: 148 us, here 51;
// B16 H32/8 over the last 4096 keys 67 and 53).
//
// A wave takes 32 keys at a time on its own, no barrier: K and V rows come by global_load_lds into its two
// buffers, whole rows by neighbouring lanes, their 16-byte chunks xored with the row so that neither the reads of
// rows (S^T = K Q^T, keys x heads) nor the transposed ones (O^T = V^T P^T) meet in a bank.  P enters as two bf16
// terms, carried to 2^-17; in v_mfma_f32_16x16x32_bf16's layouts a lane holds a head's scores of keys
// 4 (l / 16) + 0..3 of both 16-key halves, which is what the second product takes.
DEVI f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
constexpr int kTile = 32, kHeads = 16;

template <int D>
struct RowTile {  // kTile rows of D bf16
    static constexpr int C = D / 8;  // chunks per row
    u32x4 x[kTile * C];
    // The slot of chunk c of row r: rows of 256 bytes start in the same bank, of 128 in every other.
    DEVI static int slot(int r, int c) { return r * C + (c ^ (D >= 128 ? 2 * (r & 7) : D == 64 ? 2 * ((r >> 1) & 3) : 2 * ((r >> 2) & 1))); }
};

template <int D>
__global__ __launch_bounds__(kThreads) void window_decode_mfma_kernel(WinDecodeArgs a) {
    constexpr int C = D / 8, KST = D / 32, NDT = D / 16, ROWS = 64 / C;  // rows per transfer
    struct Buffers {
        RowTile<D> k[kWaves][2], v[kWaves][2];
    };
    struct Ends {  // of the waves: outputs, maxima and sums
        float o[kWaves][kHeads][D], m[kWaves][kHeads], sum[kWaves][kHeads];
    };
    union Smem {
        Buffers b;
        Ends e;
    };
    __shared__ Smem sm;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lh = lane & 15, g = lane >> 4;
    const int nhb = (a.repeat + kHeads - 1) / kHeads;
    int w = blockIdx.x;
    const int piece = w % a.splits;
    w /= a.splits;
    const int hb = w % nhb;
    w /= nhb;
    const int hk = w % a.Hkv, b = w / a.Hkv;
    const int h0 = hk * a.repeat + hb * kHeads, nh = min(kHeads, a.repeat - hb * kHeads);
    const Seen seen = seen_by(a, b);
    const int j0 = (int)((int64_t)piece * seen.n / a.splits), j1 = (int)((int64_t)(piece + 1) * seen.n / a.splits);
    const __bf16 *kb = static_cast<const __bf16 *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const __bf16 *vb = static_cast<const __bf16 *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const __bf16 *qb = static_cast<const __bf16 *>(a.q) + b * a.qs[0] + h0 * a.qs[1];
    RowTile<D>(&kt)[2] = sm.b.k[wave], (&vt)[2] = sm.b.v[wave];

    // Chunks past E are never written by a transfer: zero, once.
    if (a.E < D) {
        for (int i = lane; i < kTile * C; i += 64)
#pragma unroll
            for (int x = 0; x < 2; ++x) kt[x].x[i] = vt[x].x[i] = u32x4{0u, 0u, 0u, 0u};
        wait_lds();
    }
    // Keys j .. j + 31 on their way into buffer x (past the end: the last one again, with nothing of it).
    const int tr = lane / C, tc = lane % C;  // this lane's row and slot within a transfer
    auto start = [&](int j, int x) {
#pragma unroll
        for (int t = 0; t < kTile / ROWS; ++t) {
            const int r = t * ROWS + tr, c = RowTile<D>::slot(r, tc) - r * C;
            const int64_t key = seen.key(min(j + r, j1 - 1));
            if (8 * c < a.E) {
                lds_dma16(kb + key * a.ks[2] + 8 * c, kt[x].x + t * 64);
                lds_dma16(vb + key * a.vs[2] + 8 * c, vt[x].x + t * 64);
            }
        }
    };
    const int first = j0 + wave * kTile;
    if (first < j1) start(first, 0);
    bf16x8 qf[KST];
#pragma unroll
    for (int st = 0; st < KST; ++st) qf[st] = Ops<__bf16>::load<true>(qb + lh * a.qs[1], 32 * st + 8 * g, a.E, lh < nh);
    f32x4 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_part = 0.f;
    // What a lane reads of the tile: row lh's chunks of both halves, and for the transposed reads
    // row 4 g + lh / 4, dims 4 (lh % 4) + 0..3 of 16.
    const int vr = 4 * g + (lh >> 2);

    for (int j = first, x = 0; j < j1; j += kWaves * kTile, x ^= 1) {
        wait_vmem();
        if (j + kWaves * kTile < j1) start(j + kWaves * kTile, x ^ 1);
        float s[8];
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < KST; ++st)
                c = mfma16(__builtin_bit_cast(bf16x8, kt[x].x[RowTile<D>::slot(16 * h + lh, 4 * st + g)]), qf[st], c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[4 * h + i] = j + 16 * h + 4 * g + i < j1 ? c[i] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[4 * h + i]);
            }
        }
        // The head's maximum over the four lanes that hold its keys.
        {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = xor32_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
        }
        if (__any(mx > m_run + 8.f)) {
            const float m_new = fmaxf(m_run, mx), alpha = exp2_fast(m_run - (m_new == -INFINITY ? 0.f : m_new));
            l_part *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
            m_run = m_new;
        }
        const float ref = (m_run == -INFINITY ? 0.f : m_run) + kShift;
        u32x4 ph, pl;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p0 = exp2_fast(s[2 * i] - ref), p1 = exp2_fast(s[2 * i + 1] - ref);
            l_part += p0 + p1;
            ph[i] = cvt_pk_bf16(p0, p1);
            pl[i] = cvt_pk_bf16(p0 - __uint_as_float(ph[i] << 16), p1 - __uint_as_float(ph[i] & 0xffff0000u));
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const int c = 2 * dt + ((lh & 3) >> 1);
            const char *p0 = reinterpret_cast<const char *>(&vt[x].x[RowTile<D>::slot(vr, c)]) + 8 * (lh & 1);
            const char *p1 = reinterpret_cast<const char *>(&vt[x].x[RowTile<D>::slot(16 + vr, c)]) + 8 * (lh & 1);
            const s16x4 cat[2] = {
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p0)),
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p1))};
            const bf16x8 v = __builtin_bit_cast(bf16x8, cat);
            acc[dt] = mfma16(v, __builtin_bit_cast(bf16x8, pl), acc[dt]);
            acc[dt] = mfma16(v, __builtin_bit_cast(bf16x8, ph), acc[dt]);
        }
        wait_lds();  // every read of this buffer is done before the next transfer into it
    }
    float sum = l_part;
    {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = xor32_add(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    }
    // A sum that is not finite (an infinite value seen: hi and lo terms of it cancel to NaN) is formed again below.
    float test = sum * 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) test = fmaf(acc[dt][i], 0.f, test);
    const uint64_t wrong = __ballot(lh < nh && test != 0.f);
    uint32_t again = (uint32_t)(wrong | wrong >> 16 | wrong >> 32 | wrong >> 48) & 0xffffu;
    wait_vmem();
    __syncthreads();  // every wave is done with its buffers, which the ends now take
    if (lh < nh && !((again >> lh) & 1)) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sm.e.o[wave][lh][16 * dt + 4 * g + i] = acc[dt][i];
        if (g == 0) sm.e.m[wave][lh] = m_run, sm.e.sum[wave][lh] = sum;
    }
    for (; again; again &= again - 1) {  // a head again in plain float32: lanes are keys, then dims
        const int r = __builtin_ctz(again);
        const __bf16 *q = qb + r * a.qs[1];
        auto score = [&](int j) {
            return lane < kTile && j + lane < j1
                       ? plain_dot<__bf16>(q, kb + (int64_t)seen.key(j + lane) * a.ks[2], a.E) * a.scale_log2 : -INFINITY;
        };
        float top = -INFINITY, t = 0.f, o[2] = {0.f, 0.f};
        for (int j = first; j < j1; j += kWaves * kTile) top = fmaxf(top, wave_max(score(j)));
        const float ref = (top == -INFINITY ? 0.f : top) + kShift;
        for (int j = first; j < j1; j += kWaves * kTile) {
            const float p = lane < kTile && j + lane < j1 ? exp2_fast(score(j) - ref) : 0.f;
            t += wave_sum(p);
            for (int y = 0; y < min(kTile, j1 - j); ++y) {
                const float py = __shfl(p, y, 64);
                const __bf16 *v = vb + (int64_t)seen.key(j + y) * a.vs[2];
                if (lane < a.E) o[0] = fmaf(py, bf16_to_f32(v[lane]), o[0]);
                if (lane + 64 < a.E) o[1] = fmaf(py, bf16_to_f32(v[lane + 64]), o[1]);
            }
        }
        if (lane < D) sm.e.o[wave][r][lane] = o[0];
        if (lane + 64 < D) sm.e.o[wave][r][lane + 64] = o[1];
        if (lane == 0) sm.e.m[wave][r] = top, sm.e.sum[wave][r] = t;
    }
    __syncthreads();
    for (int i = tid; i < nh * D; i += kThreads) join_waves<__bf16>(a, &sm.e.o[0][0][0], &sm.e.m[0][0], &sm.e.sum[0][0], kHeads, D, b, h0, piece, i / D, i % D);
}

// Joins the pieces of a row, a wave each: lanes are pieces for the maximum and sum, then dims.
template <typename T>
__global__ __launch_bounds__(64) void window_decode_merge_kernel(WinDecodeArgs a) {
    const int64_t row = blockIdx.x;
    const float *part = a.part + row * a.splits * (a.E + 2);
    const int lane = threadIdx.x;
    float top = -INFINITY, t = 0.f;
    for (int i = lane; i < a.splits; i += 64) top = fmaxf(top, part[i * (a.E + 2) + a.E]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int i = lane; i < a.splits; i += 64) t = fmaf(exp2_fast(part[i * (a.E + 2) + a.E] - ref), part[i * (a.E + 2) + a.E + 1], t);
    t = wave_sum(t);
    const float inv = t == 0.f ? 0.f : 1.f / t;
    for (int d = lane; d < a.E; d += 64) {
        float o = 0.f;
#pragma unroll 4
        for (int i = 0; i < a.splits; ++i) o = fmaf(exp2_fast(part[i * (a.E + 2) + a.E] - ref) * inv, part[i * (a.E + 2) + d], o);
        static_cast<T *>(a.out)[row * a.E + d] = from_f32<T>(o);
    }
    if (lane == 0) a.lse[row] = t == 0.f ? 0.f : (ref + kShift + log2_fast(t)) * kLn2;
}

// The heads that share a row's registers: float32 B8, 8 kv heads, 4096 keys with 8 heads each 80 us, and 171 with a
// workgroup per head; 4 heads 58 and 86.
int heads_per_block(int repeat) { return repeat >= 5 ? 8 : repeat >= 3 ? 4 : repeat; }

bool on_mfma(const WinDecodeArgs &a, bool bf16) { return bf16 && a.vec && a.E <= 128; }

template <int D>
hipError_t launch_mfma(const WinDecodeArgs &a, hipStream_t st) {
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.repeat + kHeads - 1) / kHeads) * a.splits;
    return launch(window_decode_mfma_kernel<D>, dim3((unsigned)blocks), dim3(kThreads), st, a);
}

template <typename T, int LPR, int REP, bool VEC>
hipError_t launch_r(const WinDecodeArgs &a, hipStream_t st) {
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.repeat + REP - 1) / REP) * a.splits;
    return launch(window_decode_kernel<T, LPR, REP, VEC>, dim3((unsigned)blocks), dim3(kThreads), st, a);
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

// Pieces of a sequence's keys, of at least 128: as many as give every CU one workgroup of the MFMA kernel, whose
// buffers fill its LDS (with two of them in turn B16 H32/8 E128 over the last 4096 keys takes 60 us and not 57, B2 with
// 8192 keys 27 and not 21), and two of the other (float32 B8 H32/8, 4096 keys: 64 us with one, 51 with two, 58
// with four).
int window_decode_splits(const WinDecodeArgs &a, bool bf16) {
    const int per = on_mfma(a, bf16) ? kHeads : heads_per_block(a.repeat);
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.repeat + per - 1) / per);
    const int64_t span = std::min<int64_t>(a.S, (int64_t)a.window + a.sinks), cus = std::max(device_cus(), 1);
    if (blocks == 0) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(span / 128, (on_mfma(a, bf16) ? 1 : 2) * cus / blocks));
}

hipError_t launch_window_decode(const WinDecodeArgs &a, bool bf16, hipStream_t st) {
    if (on_mfma(a, bf16)) {
        if (a.E <= 32) return_if(launch_mfma<32>(a, st));
        else if (a.E <= 64) return_if(launch_mfma<64>(a, st));
        else return_if(launch_mfma<128>(a, st));
    } else if (bf16) {
        return_if((a.vec ? launch_v<__bf16, true>(a, st) : launch_v<__bf16, false>(a, st)));
    } else {
        return_if((a.vec ? launch_v<float, true>(a, st) : launch_v<float, false>(a, st)));
    }
    if (a.splits == 1) return hipSuccess;
    const dim3 grid((unsigned)((int64_t)a.B * a.H)), block(64);
    return bf16 ? launch(window_decode_merge_kernel<__bf16>, grid, block, st, a)
                : launch(window_decode_merge_kernel<float>, grid, block, st, a);
}

}  // namespace dc
