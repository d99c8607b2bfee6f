// Attention with a sliding window and sinks (dc_window.h): parameter block, launchers, and what the
// forward and backward kernels share: which key tiles a block of queries reads, operand fragments of
// both types and tiles of rows in LDS.
//
// One source for both types.  float32 operands are split exactly into three bf16 parts (x3.hpp), six
// products each, error below the float32 MFMA's.  bf16 operands enter the MFMAs as they are, and what the
// kernels compute (P, dS) as two bf16 terms hi + lo, carried to 2^-17.  So neither type has a rounding to
// fewer bits before the result's own.  (bf16 without the lo terms wherever every P of a block is below
// 1/32: a training step of B2 H32/8 L8192 E128 W1024 takes 1738 us and not 1999, but its gradients are
// 2.2e-3 from float64 by norm and not 1.7e-3, which is the rounding of the results alone.)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"
#include "tile_bf16.hpp"
#include "x3.hpp"

namespace dc {

struct WinArgs {
    int B, H, Hkv, L, S, E, repeat;
    int offset, window, sinks;
    float scale, scale_log2;  // natural and base 2
    const void *q, *k, *v, *dout, *out_in;
    const float *lse_in;
    int64_t qs[3], ks[3], vs[3], gs[3];  // strides: batch, head, row
    void *out;
    void *rest;           // bf16, optional: what rounding out left, itself rounded (forward: written, backward: read)
    float *lse;
    void *dq, *dk, *dv;
    float *dsum;          // (B, H, L): rowsum(dO * O)
    // dK / dV: the first sink_tiles key tiles (those that hold sinks: every later query sees them) run
    // as sink_pieces pieces of their queries, the others as tile_pieces, each leaving float32 partials
    // in kv_part (1: results directly).
    int sink_tiles, sink_pieces, tile_pieces;
    float *kv_part;
    bool pack;            // forward: rows of all the heads of a kv head share tiles
    int splits;           // forward: pieces of each tile's keys
    float *part, *part_lse;
    bool vec;             // 16-byte pieces: rows and bases on 16 bytes, E a whole number of pieces
};

hipError_t launch_window_fwd(const WinArgs &a, bool bf16, size_t part_bytes, hipStream_t st);
size_t window_fwd_part_bytes(const WinArgs &a, bool bf16);
hipError_t launch_window_bwd(const WinArgs &a, bool bf16, hipStream_t st);
size_t window_bwd_part_bytes(const WinArgs &a, bool bf16);  // of kv_part

struct WinDecodeArgs {
    int B, H, Hkv, S, E, repeat;
    int window, sinks;
    float scale_log2;
    const void *q, *k, *v, *lengths;
    int length_bytes;
    int64_t qs[3], ks[3], vs[3];
    void *out;
    float *lse;
    float *part;
    int splits;
    bool vec;
};
hipError_t launch_window_decode(const WinDecodeArgs &a, bool bf16, hipStream_t st);
int window_decode_splits(const WinDecodeArgs &a, bool bf16);

namespace {

// Whether the query at position p sees key s (s < S is the caller's).
DEVI bool sees(int p, int s, int window, int sinks) { return s <= p && (p - s < window || s < sinks); }

// Whether it sees any key at all.
DEVI bool sees_any(const WinArgs &a, int p) { return a.S > 0 && (a.sinks > 0 || p - a.window < a.S - 1); }

// Which of the keys base + c a query at p sees (c a constant): three compares, no branch.
struct SeenKeys {
    int hi, lo, sink;
    DEVI SeenKeys(int p, int base, int S, int window, int sinks)
        : hi(min(p, S - 1) - base), lo(max(p - window, -1) - base), sink(sinks - base) {}
    DEVI bool operator()(int c) const { return (c <= hi) & ((c > lo) | (c < sink)); }
};
// And which of the queries at base + c see a key.
struct SeenBy {
    int first, end;
    DEVI SeenBy(int key, int base, int S, int window, int sinks) : first(key < S ? key - base : 64) {
        const int64_t e = (int64_t)key + window - base;
        end = key < sinks || e > 64 ? 64 : (int)max(e, (int64_t)-64);
    }
    DEVI bool operator()(int c) const { return (c >= first) & (c < end); }
};
constexpr int acc_const(int e) { return 8 * (e >> 2) + (e & 3); }  // acc_row without its 4 g

// The key tiles (of BN keys) that queries at positions p0 .. p1 read: ns tiles from key 0 (sinks), then
// those from tile tb; n in all.  One run from tile 0 where the two meet.
struct Band {
    int ns, tb, n;
    __host__ __device__ int tile(int i) const { return i < ns ? i : tb + (i - ns); }
};
__host__ __device__ inline Band band_of(int p0, int p1, int S, int window, int sinks, int BN) {
    const int hi = p1 < S - 1 ? p1 + 1 : S;           // keys below hi
    const int lo = p0 >= window ? p0 - window + 1 : 0;  // and from lo on, or below sinks
    const int sink_end = sinks < hi ? sinks : hi;
    Band b;
    b.ns = (sink_end + BN - 1) / BN;
    b.tb = lo / BN;
    int te = lo < hi ? (hi + BN - 1) / BN : b.tb;
    if (b.ns > 0 && b.ns >= b.tb) {  // meet: one run
        if (te < b.ns) te = b.ns;
        b.ns = 0, b.tb = 0;
    }
    b.n = b.ns + (te - b.tb);
    return b;
}

#define lds __attribute__((address_space(3)))  // pointers into LDS

// Operands of one type.
template <typename T>
struct Ops;
template <>
struct Ops<__bf16> {
    typedef bf16x8 Frag;
    template <int R, int D>
    struct Tile {
        u32x4 p[CMTile<R, D>::SLOTS];
    };
    template <int R, int D>
    DEVI static Frag row(const Tile<R, D> &t, uint32_t base, int row0, int st) { return row_frag<R, D>(t.p, base, row0, st); }
    template <int R, int D>
    DEVI static Frag tr(const Tile<R, D> &t, uint32_t base, int row0, int dt) { return tr_frag<R, D>(t.p, base, row0, dt); }
    static constexpr int READS = 1, MMAS = 1;  // 16-byte LDS reads of a row fragment, MFMAs of a product
    DEVI static f32x16 mma(Frag a, Frag b, f32x16 c) { return mfma_bf16(a, b, c); }
    // c[i] += a[i] x[at .. at + 7], the N independent chains product by product.
    template <int N>
    DEVI static void mma_p(const Frag (&a)[N], const f32x16 &x, int at, f32x16 (&c)[N]) {
        Frag h, l;
        split_bf16(x, at, h, l);
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = mfma_bf16(a[i], l, c[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = mfma_bf16(a[i], h, c[i]);
    }
    // Dims d0 .. d0 + 7 of a row (0 past E, and all 0 without `in`).
    template <bool VEC>
    DEVI static Frag load(const __bf16 *row, int d0, int E, bool in) {
        Frag f;
        if (VEC) {
            const u32x4 z = {0u, 0u, 0u, 0u};
            f = __builtin_bit_cast(bf16x8, in && d0 < E ? *reinterpret_cast<const u32x4 *>(row + d0) : z);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = in && d0 + e < E ? row[d0 + e] : static_cast<__bf16>(0.f);
        }
        return f;
    }
    DEVI static Frag neg(Frag f) {
        u32x4 x = __builtin_bit_cast(u32x4, f);
        x ^= 0x80008000u;
        return __builtin_bit_cast(bf16x8, x);
    }
    // a . b of two fragments' own 8 dims.
    DEVI static float dot(Frag a, Frag b) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(bf16_to_f32(a[e]), bf16_to_f32(b[e]), s);
        return s;
    }
};
template <>
struct Ops<float> {
    typedef X3 Frag;
    template <int R, int D>
    using Tile = X3Tile<R, D>;
    template <int R, int D>
    DEVI static Frag row(const Tile<R, D> &t, uint32_t base, int row0, int st) { return row_frag_x3<R, D>(t, base, row0, st); }
    template <int R, int D>
    DEVI static Frag tr(const Tile<R, D> &t, uint32_t base, int row0, int dt) { return tr_frag_x3<R, D>(t, base, row0, dt); }
    static constexpr int READS = 3, MMAS = 6;
    DEVI static f32x16 mma(const Frag &a, const Frag &b, f32x16 c) { return mfma_x3(a, b, c); }
    template <int N>
    DEVI static void mma_p(const Frag (&a)[N], const f32x16 &x, int at, f32x16 (&c)[N]) {
        const X3 p = split3(x, at);
#pragma unroll
        for (int j = 0; j < 6; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = mfma_x3_part(a[i], p, c[i], j);
    }
    template <bool VEC>
    DEVI static Frag load(const float *row, int d0, int E, bool in) {
        f32x4 x[2];
        load_chunk<VEC>(x, row, d0, in ? E : 0);
        return split_chunk(x);
    }
    DEVI static Frag neg(const Frag &f) { return {Ops<__bf16>::neg(f.h), Ops<__bf16>::neg(f.m), Ops<__bf16>::neg(f.l)}; }
    DEVI static float dot(const Frag &a, const Frag &b) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            s = fmaf((bf16_to_f32(a.l[e]) + bf16_to_f32(a.m[e])) + bf16_to_f32(a.h[e]),
                     (bf16_to_f32(b.l[e]) + bf16_to_f32(b.m[e])) + bf16_to_f32(b.h[e]), s);
        return s;
    }
};

// R rows of D dims on their way from memory (row stride `ld`) into an LDS tile by THREADS threads: start()
// issues the loads, finish() ends them (the caller then synchronizes).  Rows from `rows` on and dims
// past E are 0.
//
// bf16 in 16-byte pieces: global_load_lds, lane l taking row l of a 64-row block, no registers between.
// Dims past E are zeroed once for the kernel's life by clear() (no transfer writes there).  Otherwise,
// and float32 (split on the way), through registers.
template <typename T, int R, int D, int THREADS, bool VEC>
struct Stage;
template <int R, int D, int THREADS>
struct Stage<__bf16, R, D, THREADS, true> {
    typedef Ops<__bf16>::Tile<R, D> Tile;
    DEVI static void clear(Tile &t, int E, int tid) {
        for (int i = (E / 8) * CMTile<R, D>::P + tid; i < CMTile<R, D>::SLOTS; i += THREADS) t.p[i] = u32x4{0u, 0u, 0u, 0u};
    }
    DEVI void start(Tile &t, const __bf16 *src, int64_t ld, int rows, int E, int tid) {
        static_assert(R % 64 == 0 || R == 32, "64 rows at a time, or half a wave's");
        constexpr int W = THREADS / 64, RB = R / 64 ? R / 64 : 1, NT = CMTile<R, D>::C * RB, count = (NT + W - 1) / W;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
        const uint32_t loff = (uint32_t)lane * (uint32_t)(ld * 2);
        // Transfer x moves chunk x / RB of rows 64 (x % RB) + lane.
        if (R >= 64 && NT % (2 * W) == 0 && rows >= R && E == D) {
            // Whole tiles in straight lines, two transfers a statement: their tests and address arithmetic are a
            // wave's own time (forward B2 H32/8 L8192 E128 W1024 459 -> 444 us, B4 H32 L4096 E64 279 -> 262).
            const uint32_t to = (uint32_t)(uintptr_t)(const lds u32x4 *)t.p;
            const uint64_t from = sgpr_addr(src), block = sgpr_addr(src + 64 * ld) - from;
#pragma unroll
            for (int j = 0; j < count; j += 2) {
                const int x = wave + W * j, y = x + W;
                const uint64_t gx = from + 16 * (x / RB) + x % RB * block, gy = from + 16 * (y / RB) + y % RB * block;
                const uint32_t lx = to + 16 * (x / RB * CMTile<R, D>::P + 64 * (x % RB));
                const uint32_t ly = to + 16 * (y / RB * CMTile<R, D>::P + 64 * (y % RB));
                lds_dma16_pair(gx, loff, lx, gy, loff, ly);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < count; ++j) {
            const int inst = wave + W * j, c = inst / RB, rb = inst % RB;
            if (inst >= NT || 8 * c >= E) continue;  // wave-uniform
            u32x4 *d = t.p + c * CMTile<R, D>::P + 64 * rb;
            const int row = 64 * rb + lane;
            if (row < R) {
                if (row < rows) lds_dma16_off(src + (int64_t)(64 * rb) * ld + 8 * c, loff, d);
                else d[lane] = u32x4{0u, 0u, 0u, 0u};
            }
        }
    }
    DEVI void finish(Tile &, int) { wait_vmem(); }
};
template <int R, int D, int THREADS>
struct Stage<__bf16, R, D, THREADS, false> {
    typedef Ops<__bf16>::Tile<R, D> Tile;
    static constexpr int C = D / 8, N = (R * C + THREADS - 1) / THREADS;
    bf16x8 x[N];
    DEVI static void clear(Tile &, int, int) {}
    DEVI void start(Tile &, const __bf16 *src, int64_t ld, int rows, int E, int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = tid + THREADS * j, r = i / C, c = i % C;
            x[j] = Ops<__bf16>::load<false>(src + (int64_t)min(r, rows - 1) * ld, 8 * c, E, r < rows);
        }
    }
    DEVI void finish(Tile &t, int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = tid + THREADS * j, r = i / C, c = i % C;
            if (i < R * C) t.p[c * CMTile<R, D>::P + r] = __builtin_bit_cast(u32x4, x[j]);
        }
    }
};
template <int R, int D, int THREADS, bool VEC>
struct Stage<float, R, D, THREADS, VEC> {
    typedef Ops<float>::Tile<R, D> Tile;
    typedef X3Stage<R, D, THREADS, VEC> X;
    X s;
    DEVI static void clear(Tile &, int, int) {}
    DEVI void start(Tile &, const float *src, int64_t ld, int rows, int E, int tid) {
#pragma unroll
        for (int j = 0; j < X::N; ++j) {
            int r, c;
            X::place(j, tid, r, c);
            if (X::TOTAL % THREADS != 0 && tid + THREADS * j >= X::TOTAL) return;
            load_chunk<VEC>(s.x[j], src + (int64_t)min(r, rows - 1) * ld, 8 * c, r < rows ? E : 0);
        }
    }
    DEVI void finish(Tile &t, int tid) { s.store(t, tid); }
};

// Scheduling hint for a straight run of N steps of M MFMAs, each step consuming R LDS reads: the reads are
// kept AHEAD steps in front of their use.
template <int N, int M, int R, int AHEAD>
DEVI void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, R * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, M * AHEAD, 0);
}

// The products that form x come before what follows in program order: the compiler places them by their
// first use, behind scheduling hints and barriers, and then all of their operands' reads before them.
DEVI void pin(f32x16 &x) { asm volatile("" : "+v"(x)); }

// Four consecutive dims of a row of a result.
template <typename T, bool VEC>
DEVI void store4(T *row, int d, int E, float x0, float x1, float x2, float x3) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    if (VEC) {
        if (d < E) *reinterpret_cast<vec4 *>(row + d) = vec4{from_f32<T>(x0), from_f32<T>(x1), from_f32<T>(x2), from_f32<T>(x3)};
    } else {
        const float x[4] = {x0, x1, x2, x3};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (d + u < E) row[d + u] = from_f32<T>(x[u]);
    }
}

// A wave's 32 rows of results, value(dt, e) of its lanes' accumulators (rows on lanes), to the rows that row(r) gives (null:
// none), turned in LDS so that neighbouring lanes write neighbouring 16-byte pieces.  `room`: kRoom<D> pieces, the wave's own.
// A lane's own 8 bytes of each row otherwise: B2 H32/8 L8192 E128 W1024 forward with the rest 532 us, turned 515; W128 229 and
// 207, dQ 313 and 302; at E64 and below it takes as long or longer, and in dK / dV the registers (1023 and 1151).
template <typename T, int D, bool VEC>
constexpr bool kTurned = sizeof(T) == 2 && D == 128 && VEC;
template <int D>
constexpr int kRoom = 32 * (D / 8 + 1);
template <int D, typename Value, typename Row>
DEVI void store_turned(u32x4 *room, int lane, int E, Value value, Row row) {
    constexpr int C = D / 8, P = C + 1;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            reinterpret_cast<u32x2 *>(room + (lane & 31) * P + 4 * dt + e / 4)[lane >> 5] =
                u32x2{cvt_pk_bf16(value(dt, e), value(dt, e + 1)), cvt_pk_bf16(value(dt, e + 2), value(dt, e + 3))};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
        const int r = (64 * i + lane) / C, c = (64 * i + lane) % C;
        __bf16 *to = row(r);
        if (to && 8 * c < E) *reinterpret_cast<u32x4 *>(to + 8 * c) = room[r * P + c];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the room is written again
}

// What rounding x to bf16 leaves.
DEVI float rest_of(float x) { return x - bf16_to_f32(f32_to_bf16(x)); }

// a . b over E dims in plain float32, for rows computed again.
template <typename T>
DEVI float plain_dot(const T *a, const T *b, int E) {
    float s = 0.f;
    for (int d = 0; d < E; ++d) s = fmaf(to_f32<T>(a[d]), to_f32<T>(b[d]), s);
    return s;
}

// Whether a row's E dims, in lanes' x0 and x1 (dims lane and lane + 64), are all NaN: nothing added changes them.
DEVI bool all_nan(int lane, int E, float x0, float x1) {
    return __all((lane >= E || x0 != x0) && (lane + 64 >= E || x1 != x1));
}

DEVI float wave_max(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
DEVI float wave_sum(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

}  // namespace
}  // namespace dc
