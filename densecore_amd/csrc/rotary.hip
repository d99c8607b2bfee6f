// Position rotation of queries and keys, alone or behind a root-mean-square norm of each head, and
// its gradient (dc_rotary.h).
//
// A row (one head of one token, E dims) belongs to a group of G lanes.  A lane owns a unit: V pairs,
// that is two 16-byte pieces of the row, (i, i + R/2) or the 2 V consecutive dims of V interleaved
// pairs; the dims behind the rotated ones are units whose angle is 0.  So both members of a pair are
// in one lane, the norm's sum is a butterfly over the group, and a row is read and written once.
//
// Angles: a = p f in float64, in quarter turns t = p f 2/pi; t - rint(t) is exact, so the argument left
// for sine and cosine is at most pi/4 with an error of p f 2^-52, whatever the position (float32 angles
// are wrong by 2^-4 at a position of 2^20).  Both are then Taylor sums in float32 (below).  A group keeps
// its token's angles over `hb` heads, so they cost a tenth of the loads' time.
//
// Bound: HBM, each value in and out once (the norm's gradient reads x again).  B2 H32/8 L8192 E128 bf16: rotation
// 66 us (335 MB, 5.1 TB/s; a copy of 2 GiB runs at 4.86), with norm 68, the norm's gradient 104 (503 MB, 4.8
// TB/s).  One token: 4 us, a launch's latency.
#include <algorithm>

#include "common.hpp"
#include "params.hpp"
#include "rotary.hpp"

namespace dc {
namespace {

constexpr int kThreads = 256;

// cos and sin of quarter turns `t`, times m.  |x| <= pi/4: the Taylor sums to x^9 and x^10 are off by
// x^11 / 11! < 1.8e-9 and x^12 / 12! < 1.2e-10, a fortieth of a float32 rounding.
DEVI void turn_of(double t, float m, float &c, float &s) {
    const double q = rint(t);
    const float x = (float)((t - q) * 1.57079632679489662);
    const int quad = (int)(q - 4.0 * floor(q * 0.25));
    const float z = x * x;
    float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(z, sn, 8.3333333e-3f);
    sn = fmaf(z, sn, -1.6666667e-1f);
    sn = fmaf(z * x, sn, x);
    float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    cs = fmaf(z, cs, -1.3888889e-3f);
    cs = fmaf(z, cs, 4.1666667e-2f);
    cs = fmaf(z, cs, -0.5f);
    cs = fmaf(z, cs, 1.f);
    const float a = (quad & 1) ? sn : cs, b = (quad & 1) ? cs : sn;
    c = ((quad == 1 || quad == 2) ? -a : a) * m;
    s = ((quad & 2) ? -b : b) * m;
}

// V consecutive values, one store where V > 1 (the launcher checks the alignment).
template <typename T, int V>
DEVI void store_v(T *p, const float (&x)[V]) {
    if constexpr (V == 1) {
        *p = from_f32<T>(x[0]);
    } else {
        typedef T vec __attribute__((ext_vector_type(V)));
        vec r;
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = from_f32<T>(x[e]);
        *reinterpret_cast<vec *>(p) = r;
    }
}

// Where unit u's two pieces start (b == E: there is no second piece), and whether it is rotated.
struct Unit {
    int a, b;
    bool in, turned;
};
template <int V>
DEVI Unit unit_of(int u, int E, int R, bool interleaved) {
    const int P = R / 2, turned = P / V, rest = (E - R + 1) / 2;
    if (u < turned) return interleaved ? Unit{2 * u * V, 2 * u * V + V, true, true} : Unit{u * V, P + u * V, true, true};
    const int t = (u - turned) * V;
    return {R + t, min(R + rest + t, E), t < rest, false};
}

// A lane's pieces of a row as they lie (loads in flight cost no more registers than that), and as float32.
template <typename T, int V, int NU>
struct RowRaw {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec a[NU], b[NU];
    // (Pieces a lane does not have are 0.)
    DEVI void load(const T *row, const Unit (&un)[NU], int E, bool in) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const bool ina = in && un[i].in, inb = ina && (V > 1 || un[i].b < E);
            a[i] = ina ? *reinterpret_cast<const vec *>(row + un[i].a) : vec(T(0));
            b[i] = inb ? *reinterpret_cast<const vec *>(row + un[i].b) : vec(T(0));
        }
    }
};
template <typename T, int V, int NU>
struct RowVals {
    float a[NU][V], b[NU][V];
    DEVI void set(const RowRaw<T, V, NU> &r) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) a[i][e] = to_f32<T>(r.a[i][e]), b[i][e] = to_f32<T>(r.b[i][e]);
    }
    DEVI void store(T *row, const Unit (&un)[NU], int E) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            if (un[i].in) store_v<T, V>(row + un[i].a, a[i]);
            if (un[i].in && (V > 1 || un[i].b < E)) store_v<T, V>(row + un[i].b, b[i]);
        }
    }
};

// Cosines and sines of a lane's pairs (1 and 0 where the dims are not rotated).
template <int V, int NU>
struct Angles {
    float c[NU][V], s[NU][V];
    DEVI void set(double p, const RotArgs &a, int lane_u, int G, const Unit (&un)[NU]) {
        typedef double vec __attribute__((ext_vector_type(V)));
        p *= 0.63661977236758134;  // quarter turns
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const vec f = un[i].turned ? *reinterpret_cast<const vec *>(a.freq + (lane_u + i * G) * V) : vec(0.0);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                turn_of(p * f[e], a.magnitude, c[i][e], s[i][e]);
                if (!un[i].turned) c[i][e] = 1.f, s[i][e] = 0.f;
            }
        }
    }
    // The turn (sign 1) or the turn back (sign -1) of a row's values.
    template <typename T>
    DEVI void apply(RowVals<T, V, NU> &x, const Unit (&un)[NU], bool interleaved, float sign) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            if (!un[i].turned) continue;
            if (V > 1 && interleaved) {
                float v[2 * V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = x.a[i][e], v[V + e] = x.b[i][e];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float x1 = v[2 * e], x2 = v[2 * e + 1], sn = sign * s[i][e];
                    v[2 * e] = fmaf(x1, c[i][e], -x2 * sn);
                    v[2 * e + 1] = fmaf(x2, c[i][e], x1 * sn);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) x.a[i][e] = v[e], x.b[i][e] = v[V + e];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float x1 = x.a[i][e], x2 = x.b[i][e], sn = sign * s[i][e];
                    x.a[i][e] = fmaf(x1, c[i][e], -x2 * sn);
                    x.b[i][e] = fmaf(x2, c[i][e], x1 * sn);
                }
            }
        }
    }
};

DEVI double position_of(const RotArgs &a, int64_t b, int64_t l) {
    if (a.pos_bytes == 0) return (double)(a.offset + l);
    const int64_t at = b * a.pos_sb + l * a.pos_sl;
    return a.pos_bytes == 8 ? (double)static_cast<const int64_t *>(a.pos)[at]
                            : (double)static_cast<const int32_t *>(a.pos)[at];
}

template <typename W, int V, int NU>
DEVI void load_weight_of(const W *w, const Unit (&un)[NU], int E, float (&wa)[NU][V], float (&wb)[NU][V]) {
    RowRaw<W, V, NU> raw;
    raw.load(w, un, E, true);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) wa[i][e] = to_f32<W>(raw.a[i][e]), wb[i][e] = to_f32<W>(raw.b[i][e]);
}
template <int V, int NU>
DEVI void load_weight(const void *w, bool bf16, const Unit (&un)[NU], int E, float (&wa)[NU][V], float (&wb)[NU][V]) {
    if (w && bf16) return load_weight_of<__bf16, V, NU>(static_cast<const __bf16 *>(w), un, E, wa, wb);
    if (w) return load_weight_of<float, V, NU>(static_cast<const float *>(w), un, E, wa, wb);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) wa[i][e] = wb[i][e] = 1.f;
}

// Forward (and, with inverse and no norm, the gradient): items of (block of hb heads, token), token
// fastest, dealt to groups of G lanes.
template <typename T, int V, int G, int NU, bool NORM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotArgs a, bool inverse) {
    constexpr int HU = NU > 1 ? 2 : 4;  // rows in flight per lane
    const int lane_u = threadIdx.x % G;
    const int64_t stride = (int64_t)gridDim.x * (kThreads / G);
    const int qb = (a.t[0].heads + a.hb - 1) / a.hb, kb = (a.t[1].heads + a.hb - 1) / a.hb;
    const int64_t items = (int64_t)(qb + kb) * a.tokens;
    const float inv_e = 1.f / (float)a.E;
    Unit un[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) un[i] = unit_of<V>(lane_u + i * G, a.E, a.R, a.interleaved);
    for (int64_t item = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G; item < items; item += stride) {
        const int64_t token = item % a.tokens;
        int blk = (int)(item / a.tokens);
        const int which = blk >= qb ? 1 : 0;
        blk -= which * qb;
        const RotRows &t = a.t[which];
        const int64_t b = token / a.L, l = token % a.L;
        const int h0 = blk * a.hb, h1 = min(h0 + a.hb, t.heads);
        const T *src = static_cast<const T *>(inverse ? t.g : t.x);
        const int64_t sb = inverse ? t.gs[0] : t.xs[0], sh = inverse ? t.gs[1] : t.xs[1], sl = inverse ? t.gs[2] : t.xs[2];
        src += b * sb + l * sl;
        T *dst = static_cast<T *>(t.out) + (b * t.heads * a.L + l) * a.E;
        Angles<V, NU> ang;
        RowRaw<T, V, NU> raw[HU];
        float wa[NU][V], wb[NU][V];
        for (int h = h0; h < h1; h += HU) {
#pragma unroll
            for (int j = 0; j < HU; ++j) raw[j].load(src + (h + j) * sh, un, a.E, h + j < h1);
            if (h == h0) {  // while the first rows are on their way
                ang.set(position_of(a, b, l), a, lane_u, G, un);
                if constexpr (NORM) load_weight<V, NU>(t.w, a.w_bf16, un, a.E, wa, wb);
            }
#pragma unroll
            for (int j = 0; j < HU; ++j) {
                RowVals<T, V, NU> x;
                x.set(raw[j]);
                if constexpr (NORM) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < NU; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) ss = fmaf(x.a[i][e], x.a[i][e], fmaf(x.b[i][e], x.b[i][e], ss));
                    const float r = rsqrtf(fmaf(lanes_sum<G>(ss), inv_e, a.eps));
#pragma unroll
                    for (int i = 0; i < NU; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) x.a[i][e] *= r * wa[i][e], x.b[i][e] *= r * wb[i][e];
                }
                ang.apply(x, un, a.interleaved, inverse ? -1.f : 1.f);
                if (h + j < h1) x.store(dst + (int64_t)(h + j) * a.L * a.E, un, a.E);
            }
        }
    }
}

// Gradient with norm: with t = the gradient turned back times m, s = sum t w x,
//     dx = r (t w - x r^2 s / E),   dw = sum over rows of t x r.
// The first nblk[0] workgroups take the queries, the others the keys; each keeps dw in registers over
// its rows and leaves one partial row, summed by rotary_dw_kernel in a fixed order.
template <typename T, int V, int G, int NU>
__global__ __launch_bounds__(kThreads) void rotary_norm_bwd_kernel(RotArgs a) {
    constexpr int HU = NU > 1 ? 1 : 2;
    constexpr int PER = NU * 2 * V;
    __shared__ float red[kThreads / 64][G][PER];
    const int lane_u = threadIdx.x % G, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int which = (int)blockIdx.x >= a.nblk[0] ? 1 : 0;
    const int block = (int)blockIdx.x - which * a.nblk[0];
    const RotRows &t = a.t[which];
    const int64_t stride = (int64_t)a.nblk[which] * (kThreads / G);
    const int64_t items = (int64_t)((t.heads + a.hb - 1) / a.hb) * a.tokens;
    const float inv_e = 1.f / (float)a.E;
    Unit un[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) un[i] = unit_of<V>(lane_u + i * G, a.E, a.R, a.interleaved);
    float wa[NU][V], wb[NU][V], da[NU][V], db[NU][V];
    load_weight<V, NU>(t.w, a.w_bf16, un, a.E, wa, wb);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) da[i][e] = db[i][e] = 0.f;
    for (int64_t item = (int64_t)block * (kThreads / G) + threadIdx.x / G; item < items; item += stride) {
        const int64_t token = item % a.tokens;
        const int h0 = (int)(item / a.tokens) * a.hb, h1 = min(h0 + a.hb, t.heads);
        const int64_t b = token / a.L, l = token % a.L;
        const T *src = static_cast<const T *>(t.x) + b * t.xs[0] + l * t.xs[2];
        const T *grd = static_cast<const T *>(t.g) + b * t.gs[0] + l * t.gs[2];
        T *dst = static_cast<T *>(t.out) + (b * t.heads * a.L + l) * a.E;
        Angles<V, NU> ang;
        RowRaw<T, V, NU> xr[HU], yr[HU];
        for (int h = h0; h < h1; h += HU) {
#pragma unroll
            for (int j = 0; j < HU; ++j) {
                xr[j].load(src + (h + j) * t.xs[1], un, a.E, h + j < h1);
                yr[j].load(grd + (h + j) * t.gs[1], un, a.E, h + j < h1);
            }
            if (h == h0) ang.set(position_of(a, b, l), a, lane_u, G, un);
#pragma unroll
            for (int j = 0; j < HU; ++j) {
                RowVals<T, V, NU> x, y;
                x.set(xr[j]), y.set(yr[j]);
                ang.apply(y, un, a.interleaved, -1.f);
                float ss = 0.f, st = 0.f;
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float xa = x.a[i][e], xb = x.b[i][e];
                        ss = fmaf(xa, xa, fmaf(xb, xb, ss));
                        st = fmaf(y.a[i][e] * wa[i][e], xa, fmaf(y.b[i][e] * wb[i][e], xb, st));
                    }
                const float r = rsqrtf(fmaf(lanes_sum<G>(ss), inv_e, a.eps));
                const float k = r * r * (lanes_sum<G>(st) * inv_e);
                const bool in = h + j < h1;  // (a row of zeros with eps 0 has no r)
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float xa = x.a[i][e], xb = x.b[i][e], ya = y.a[i][e], yb = y.b[i][e];
                        if (in) da[i][e] = fmaf(ya, xa * r, da[i][e]), db[i][e] = fmaf(yb, xb * r, db[i][e]);
                        x.a[i][e] = r * fmaf(ya, wa[i][e], -xa * k);
                        x.b[i][e] = r * fmaf(yb, wb[i][e], -xb * k);
                    }
                if (in) x.store(dst + (int64_t)(h + j) * a.L * a.E, un, a.E);
            }
        }
    }
    if (!a.part[which]) return;
    // The groups of a wave, then the waves, then one row of this workgroup.
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
#pragma unroll
            for (int o = G; o < 64; o <<= 1) {
                da[i][e] += __shfl_xor(da[i][e], o, 64);
                db[i][e] += __shfl_xor(db[i][e], o, 64);
            }
            if (lane < G) red[wave][lane_u][(i * 2) * V + e] = da[i][e], red[wave][lane_u][(i * 2 + 1) * V + e] = db[i][e];
        }
    __syncthreads();
    if (threadIdx.x >= G) return;
    float *row = a.part[which] + (int64_t)block * a.E;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float sa = 0.f, sb = 0.f;
#pragma unroll
            for (int w = 0; w < kThreads / 64; ++w) sa += red[w][lane_u][(i * 2) * V + e], sb += red[w][lane_u][(i * 2 + 1) * V + e];
            if (un[i].in) row[un[i].a + e] = sa;
            if (un[i].in && un[i].b + e < a.E) row[un[i].b + e] = sb;
        }
}

// dw[d] = the sum over the workgroups' rows: 8 dims per workgroup, 32 threads per dim.
__global__ __launch_bounds__(256) void rotary_dw_kernel(RotArgs a) {
    __shared__ float red[32][9];
    const int which = blockIdx.y, d = blockIdx.x * 8 + (threadIdx.x & 7), p = threadIdx.x >> 3;
    if (!a.part[which]) return;
    float s = 0.f;
    if (d < a.E) {
#pragma unroll 8
        for (int r = p; r < a.nblk[which]; r += 32) s += a.part[which][(int64_t)r * a.E + d];
    }
    red[p][threadIdx.x & 7] = s;
    __syncthreads();
    if (p != 0 || d >= a.E) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
    if (a.w_bf16) static_cast<__bf16 *>(a.dw[which])[d] = f32_to_bf16(s);
    else static_cast<float *>(a.dw[which])[d] = s;
}

// 16-byte pieces: whole pieces of pairs and of the dims behind them, rows that start on 16 bytes.
bool pieces(const RotArgs &a, int V, int size) {
    if (a.R / 2 % V != 0 || a.E % (2 * V) != 0 || (reinterpret_cast<uintptr_t>(a.freq) & 15) != 0) return false;
    for (const RotRows &t : a.t) {
        if (t.heads == 0) continue;
        for (const void *p : {t.x, t.g, t.w, static_cast<const void *>(t.out)})
            if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) return false;
        for (int i = 0; i < 3; ++i)
            if ((t.x && t.xs[i] * size % 16 != 0) || (t.g && t.gs[i] * size % 16 != 0)) return false;
    }
    return true;
}

template <typename T, int V, int G, int NU>
hipError_t launch_g(const RotArgs &args, bool inverse, bool norm_bwd, hipStream_t st) {
    RotArgs a = args;
    constexpr int GROUPS = kThreads / G;
    const int cus = std::max(device_cus(), 1);
    const int64_t heads = a.t[0].heads + a.t[1].heads;
    // Heads one after the other with the same angles: as many as leave 2 workgroups per CU, up to 16.  H32/8 E128
    // bf16 forward with norm: B2 L8192 69 us, 151 with one head at a time; 2000 tokens 11, and 21 with 8 workgroups per
    // CU; B32 L1 6 us, and 10 with 16 heads.
    a.hb = (int)std::min<int64_t>(16, std::max<int64_t>(1, heads * a.tokens / ((int64_t)GROUPS * 2 * cus)));
    auto blocks = [&](int h) { return ((int64_t)((h + a.hb - 1) / a.hb) * a.tokens + GROUPS - 1) / GROUPS; };
    if (!norm_bwd) {
        const int64_t n = std::min<int64_t>(blocks(a.t[0].heads) + blocks(a.t[1].heads), (int64_t)1 << 20);
        const dim3 grid((unsigned)n), block(kThreads);
        return a.norm ? launch(rotary_kernel<T, V, G, NU, true>, grid, block, st, a, inverse)
                      : launch(rotary_kernel<T, V, G, NU, false>, grid, block, st, a, inverse);
    }
    for (int i = 0; i < 2; ++i) a.nblk[i] = (int)std::min<int64_t>(blocks(a.t[i].heads), kRotMaxBlocks);
    // (No rows at all: the weights' gradients are the empty sum.)
    if (a.nblk[0] + a.nblk[1] > 0)
        return_if(launch(rotary_norm_bwd_kernel<T, V, G, NU>, dim3(a.nblk[0] + a.nblk[1]), dim3(kThreads), st, a));
    if (!a.part[0] && !a.part[1]) return hipSuccess;
    return launch(rotary_dw_kernel, dim3((a.E + 7) / 8, 2), dim3(256), st, a);
}

template <typename T>
hipError_t launch_t(const RotArgs &a, bool inverse, bool norm_bwd, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (pieces(a, V, sizeof(T))) {
        const int units = a.E / (2 * V);  // up to 64
        if (units <= 4) return launch_g<T, V, 4, 1>(a, inverse, norm_bwd, st);
        if (units <= 8) return launch_g<T, V, 8, 1>(a, inverse, norm_bwd, st);
        if (units <= 16) return launch_g<T, V, 16, 1>(a, inverse, norm_bwd, st);
        return launch_g<T, V, 64, 1>(a, inverse, norm_bwd, st);
    }
    const int units = a.R / 2 + (a.E - a.R + 1) / 2;  // up to 256
    if (units <= 16) return launch_g<T, 1, 16, 1>(a, inverse, norm_bwd, st);
    if (units <= 64) return launch_g<T, 1, 64, 1>(a, inverse, norm_bwd, st);
    if (units <= 128) return launch_g<T, 1, 64, 2>(a, inverse, norm_bwd, st);
    return launch_g<T, 1, 64, 4>(a, inverse, norm_bwd, st);
}

}  // namespace

hipError_t launch_rotary(const RotArgs &a, bool bf16, bool inverse, hipStream_t st) {
    return bf16 ? launch_t<__bf16>(a, inverse, false, st) : launch_t<float>(a, inverse, false, st);
}
hipError_t launch_rotary_norm_bwd(const RotArgs &a, bool bf16, hipStream_t st) {
    return bf16 ? launch_t<__bf16>(a, false, true, st) : launch_t<float>(a, false, true, st);
}

}  // namespace dc
