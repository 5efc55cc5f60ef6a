// K24: the boundary between two transformer blocks in one pass (bf16 / fp32 activations):
//
//   n = post(h)   r = x + scale * gate * n   y = pre(r)        post, gate optional; h absent: y = pre(x)
//
// post and pre are RMS norms  v / sqrt(mean(v^2) + eps) * w  or layer norms  (v - mean) / sqrt(var + eps) * w + b.
// The gate is one row per `rpg` rows of x (1: per element, S: per sequence, M: per channel).
//
// Forward: a row is held in the registers of TPR threads between its two norms, so x and h are read and r and y written
// once.  y is the norm of the unrounded r.  Backward recomputes n and r from x and h (the same bytes as reading r, and no
// rounding in between):
//   dr = dr_in + rstd (a - rhat mean(a rhat) [- mean(a)]),  a = dy w;   dx = dr;   dn = scale gate dr;   dgate = scale n dr
//   dh = rstd_h (c - hhat mean(c hhat) [- mean(c)]),  c = dn w_post
// The sums over rows (dw, db, dgate of a shared gate) run in registers over a workgroup's rows, one fp32 partial row per
// workgroup, and a second kernel adds the partials in a fixed order: no atomics.
// Both directions are HBM-bound.  16384 rows of 4096, bf16, both norms, a gate per sequence: forward 4 streams of 134 MB in
// 96 us (5.6 TB/s), backward 6 streams in 157 + 6 us (4.9 TB/s; a copy makes 4.95).  Without the gate, widths that are no
// multiple of 16 B: 4094 100 and 157 us, 4095 (every other row begins inside a dword) 120 and 206.
#include "dtf_common.h"
#include <type_traits>

struct RnArgs {
    const void *x, *h, *gate, *w, *b, *pw, *pb;
    void *y, *r;
    float* stats;                         // [4][M]: mean, rstd of pre; mean, rstd of post
    const void *dy, *dr;                  // each may be null (no gradient arrives there)
    void *dx, *dh, *dgate;                // dh null: not wanted (or equal to dx); dgate: per element only
    float* part;                          // [parts][narr][H]
    int64_t M, rpg;
    int H, wdt, layer, narr;
    // Rows come in groups of group_rows (the rows that share a gate row; one group without): workgroup id = (group - group0)
    // * nbx + bx.  More groups than workgroups go over several launches: `add` to the sums of the launches before.
    int nbx, add;
    int64_t group0, group_rows;
    int s_w, s_b, s_pw, s_pb, s_g;        // slot of each sum in a partial row, -1: none
    float scale, eps;
};

// Element e of thread l's share of a row: vectors of 16 B.  RN_ALIGNED: rows begin and end with one.  RN_ANY: they begin
// anywhere (the hardware takes unaligned vectors), and the thread whose vector would pass the row's end takes the row's last
// 16 B, of which the elements that its neighbour has too are zero in it (a shorter load there breaks the loads in flight:
// 16384 rows of 4094, bf16, backward 398 us against 157; all by elements 950).  RN_TINY: rows shorter than a vector.
enum { RN_ALIGNED, RN_ANY, RN_TINY };
typedef u32x4 rn_any4 __attribute__((aligned(2)));
typedef unsigned int rn_any1 __attribute__((aligned(2)));

template <int DT, int MODE, int TPR, int NE>
struct RnRow {
    static constexpr int V = DT == DTF_BF16 ? 8 : 4, ESZ = 16 / V;
    typedef typename std::conditional<MODE == RN_ALIGNED, u32x4, rn_any4>::type vec;
    struct Raw {                          // as it comes from memory
        u32x4 q[NE / V];
    };
    static __device__ __forceinline__ int first(int l, int c, int H) {     // column of vector c's first element
        const int at = (c * TPR + l) * V;
        return MODE == RN_ANY ? min(at, H - V) : at;
    }
    static __device__ __forceinline__ int over(int l, int c, int H) { return (c * TPR + l) * V - (H - V); }
    static __device__ __forceinline__ int col(int l, int e, int H) { return first(l, e / V, H) + e % V; }
    static __device__ __forceinline__ bool has(int l, int e, int H) {
        return MODE == RN_ANY ? e % V >= over(l, e / V, H) : col(l, e, H) < H;
    }
    // off (elements): where the row begins, uniform in a wave -- so the address is a scalar base and a 32-bit lane offset
    static __device__ __forceinline__ void fetch(const void* base, int64_t off, int H, int l, Raw& r) {
        const char* p = reinterpret_cast<const char*>(base) + off * ESZ;
#pragma unroll
        for (int c = 0; c < NE / V; ++c) {
            r.q[c] = (u32x4){0u, 0u, 0u, 0u};
            if ((c * TPR + l) * V >= H) continue;
            if constexpr (MODE == RN_TINY) {                               // (c, l = 0, H < V)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (k < H) {
                        if constexpr (DT == DTF_F32) r.q[c][k] = reinterpret_cast<const unsigned int*>(p)[k];
                        else r.q[c][k / 2] |= (unsigned int)reinterpret_cast<const unsigned short*>(p)[k] << (k & 1) * 16;
                    }
            } else r.q[c] = *reinterpret_cast<const vec*>(p + (unsigned)(first(l, c, H) * ESZ));
        }
    }
    // what a thread does not own -> 0
    static __device__ __forceinline__ void trim(Raw& r, int H, int l) {
        if constexpr (MODE == RN_ANY) {
#pragma unroll
            for (int c = 0; c < NE / V; ++c) {
                const int n = over(l, c, H);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (DT == DTF_F32) r.q[c][k] = k >= n ? r.q[c][k] : 0u;
                    else r.q[c][k] &= 2 * k >= n ? 0xffffffffu : 2 * k + 1 >= n ? 0xffff0000u : 0u;
                }
            }
        }
    }
    static __device__ __forceinline__ void expand(const Raw& r, float (&v)[NE]) {
#pragma unroll
        for (int c = 0; c < NE / V; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DT == DTF_BF16) {
                    v[c * V + 2 * k] = __uint_as_float(r.q[c][k] << 16);
                    v[c * V + 2 * k + 1] = __uint_as_float(r.q[c][k] & 0xffff0000u);
                } else v[c * V + k] = __uint_as_float(r.q[c][k]);
            }
    }
    static __device__ __forceinline__ void row(Raw r, int H, int l, float (&v)[NE]) {
        trim(r, H, l);
        expand(r, v);
    }
    static __device__ __forceinline__ void load(const void* base, int64_t off, int H, int l, float (&v)[NE]) {
        Raw r;
        fetch(base, off, H, l, r);
        row(r, H, l, v);
    }
    static __device__ __forceinline__ void store(void* base, int64_t off, int H, int l, const float (&v)[NE]) {
        char* p = reinterpret_cast<char*>(base) + off * ESZ;
#pragma unroll
        for (int c = 0; c < NE / V; ++c) {
            u32x4 q;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DT == DTF_BF16) q[k] = pack_bf16x2(v[c * V + 2 * k], v[c * V + 2 * k + 1]);
                else q[k] = __float_as_uint(v[c * V + k]);
            }
            const int at = (c * TPR + l) * V;
            char* t = p + (unsigned)(first(l, c, H) * ESZ);
            if (at >= H) continue;
            if (MODE == RN_ALIGNED || (MODE == RN_ANY && over(l, c, H) <= 0)) *reinterpret_cast<vec*>(t) = q;
            else {                                                         // bytes from `lo` on, to `hi` (uniform)
                const int lo = MODE == RN_ANY ? (V - H % V) * ESZ : 0, hi = MODE == RN_ANY ? 16 : H * ESZ;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (4 * k >= lo && 4 * k + 4 <= hi) *reinterpret_cast<rn_any1*>(t + 4 * k) = q[k];
                    else if (4 * k >= lo && 4 * k < hi) *reinterpret_cast<unsigned short*>(t + 4 * k) = (unsigned short)q[k];
                    else if (4 * k + 2 == lo) *reinterpret_cast<unsigned short*>(t + 4 * k + 2) = (unsigned short)(q[k] >> 16);
                }
            }
        }
    }
    // a parameter row of type wdt (the activations' type or fp32)
    static __device__ __forceinline__ void param(const void* p, int wdt, int H, int l, float (&v)[NE]) {
        if (wdt == DT) load(p, 0, H, l, v);
        else {
#pragma unroll
            for (int e = 0; e < NE; ++e) v[e] = has(l, e, H) ? reinterpret_cast<const float*>(p)[col(l, e, H)] : 0.f;
        }
    }
};

// sum over a wave, in every lane: inside rows of 16 by DPP (no trip through the LDS crossbar as a shuffle makes), then
// across the four rows
__device__ __forceinline__ float rn_wave_sum(float v) {
#define RN_DPP(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    RN_DPP(0xB1);       // quad_perm 1 0 3 2
    RN_DPP(0x4E);       // quad_perm 2 3 0 1
    RN_DPP(0x141);      // row_half_mirror
    RN_DPP(0x140);      // row_mirror
#undef RN_DPP
    const int i = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

// sum of a (and of b) over the TPR threads of a row; `red` alternates between two halves, one barrier a call
template <int TPR, bool TWO>
__device__ __forceinline__ void rn_sum(float& a, float& b, float (*red)[2][16], int& flip) {
    a = rn_wave_sum(a);
    if constexpr (TWO) b = rn_wave_sum(b);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6, w0 = wave & ~(TPR / 64 - 1);
        if ((threadIdx.x & 63) == 0) {
            red[flip][0][wave] = a;
            if constexpr (TWO) red[flip][1][wave] = b;
        }
        __syncthreads();
        a = 0.f;
        if constexpr (TWO) b = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) {
            a += red[flip][0][w0 + i];
            if constexpr (TWO) b += red[flip][1][w0 + i];
        }
        flip ^= 1;
    }
}

// v -> (v - mean) * rstd in place; columns past H stay 0
template <class R, int TPR, int NE>
__device__ __forceinline__ void rn_normalise(float (&v)[NE], int H, int l, float eps, int layer, float (*red)[2][16], int& flip,
                                             float& mean, float& rstd) {
    const float inv = 1.f / (float)H;
    float s = 0.f, z = 0.f;
    mean = 0.f;
    if (layer) {
#pragma unroll
        for (int e = 0; e < NE; ++e) s += v[e];
        rn_sum<TPR, false>(s, z, red, flip);
        mean = s * inv;
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = R::has(l, e, H) ? v[e] - mean : 0.f;
    }
    s = z = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) s = fmaf(v[e], v[e], s);
    rn_sum<TPR, false>(s, z, red, flip);
    rstd = 1.f / sqrtf(s * inv + eps);
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e] *= rstd;
}

template <int DT, int MODE, int TPR, int NE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rn_fwd_kernel(RnArgs a) {
    typedef RnRow<DT, MODE, TPR, NE> R;
    constexpr int RB = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[2][2][16];
    const int l = threadIdx.x % TPR, H = a.H;
    const int64_t want = (int64_t)blockIdx.x * RB + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    const int64_t row = want < a.M ? want : a.M - 1;           // spare rows of the last workgroup redo its last, unstored
    int flip = 0;
    float v[NE], p[NE], mean, rstd;
    R::load(a.x, row * H, H, l, v);
    if (a.h) {
        float n[NE];
        R::load(a.h, row * H, H, l, n);
        if (a.pw) {
            rn_normalise<R, TPR, NE>(n, H, l, a.eps, a.layer, red, flip, mean, rstd);
            if (l == 0 && want < a.M) {
                a.stats[2 * a.M + row] = mean;
                a.stats[3 * a.M + row] = rstd;
            }
            R::param(a.pw, a.wdt, H, l, p);
#pragma unroll
            for (int e = 0; e < NE; ++e) n[e] *= p[e];
            if (a.pb) {
                R::param(a.pb, a.wdt, H, l, p);
#pragma unroll
                for (int e = 0; e < NE; ++e) n[e] += p[e];
            }
        }
        if (a.gate) {
            R::load(a.gate, row / a.rpg * H, H, l, p);
#pragma unroll
            for (int e = 0; e < NE; ++e) n[e] *= p[e];
        }
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = fmaf(a.scale, n[e], v[e]);
        if (want < a.M) R::store(a.r, row * H, H, l, v);
    }
    rn_normalise<R, TPR, NE>(v, H, l, a.eps, a.layer, red, flip, mean, rstd);
    if (l == 0 && want < a.M) {
        a.stats[row] = mean;
        a.stats[a.M + row] = rstd;
    }
    R::param(a.w, a.wdt, H, l, p);
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e] *= p[e];
    if (a.b) {
        R::param(a.b, a.wdt, H, l, p);
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] += p[e];
    }
    if (want < a.M) R::store(a.y, row * H, H, l, v);
}

// A workgroup walks its rows with the next row's loads in flight and the parameters in registers (read again per row, they
// cost a cache's latency between the two reductions).  SAME: parameters of the activations' type; else (fp32 parameters of
// bf16 activations) they are read per row.
template <int DT, int MODE, int TPR, int NE, bool LAYER, bool SAME>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rn_bwd_kernel(RnArgs a) {
    typedef RnRow<DT, MODE, TPR, NE> R;
    constexpr int NT = TPR < 256 ? 256 : TPR, RB = NT / TPR;
    __shared__ float red[2][2][16];
    __shared__ float comb[RB > 1 ? NT * NE : 1];
    const int l = threadIdx.x % TPR, slot = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR), H = a.H;
    const int64_t group = a.group0 + blockIdx.x / a.nbx;
    const int bx = blockIdx.x % a.nbx;
    const int64_t r0 = group * a.group_rows;
    const int64_t r1 = r0 + a.group_rows < a.M ? r0 + a.group_rows : a.M;
    const float inv = 1.f / (float)H;
    const bool each = a.gate && a.rpg == 1;                    // a gate row per row, streamed like x
    int flip = 0;
    float sw[NE], sb[LAYER ? NE : 1], spw[NE], spb[LAYER ? NE : 1], sg[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) sw[e] = spw[e] = sg[e] = 0.f;
    if constexpr (LAYER) {
#pragma unroll
        for (int e = 0; e < NE; ++e) sb[e] = spb[e] = 0.f;
    }
    typename R::Raw wr, pwr, pbr, gr, xr, hr, dyr, drr;
    if constexpr (SAME) {
        R::fetch(a.w, 0, H, l, wr);
        if (a.pw) R::fetch(a.pw, 0, H, l, pwr);
        if (LAYER && a.pb) R::fetch(a.pb, 0, H, l, pbr);
    }
    if (a.gate && !each) R::fetch(a.gate, r0 / a.rpg * H, H, l, gr);
    auto row_at = [&](int64_t base) { return base + slot < r1 ? base + slot : r1 - 1; };      // spare rows redo the last, unstored
    float mean = 0.f, rstd = 1.f, pmean = 0.f, prstd = 1.f;
    auto fetch = [&](int64_t row) {
        R::fetch(a.x, row * H, H, l, xr);
        if (a.h) R::fetch(a.h, row * H, H, l, hr);
        if (each) R::fetch(a.gate, row * H, H, l, gr);
        if (a.dy) R::fetch(a.dy, row * H, H, l, dyr);
        if (a.dr) R::fetch(a.dr, row * H, H, l, drr);
        if (LAYER) mean = a.stats[row];
        rstd = a.stats[a.M + row];
        if (a.pw) {
            if (LAYER) pmean = a.stats[2 * a.M + row];
            prstd = a.stats[3 * a.M + row];
        }
    };
    const int64_t first = r0 + (int64_t)bx * RB, stride = (int64_t)a.nbx * RB;
    if (first < r1) fetch(row_at(first));
    if constexpr (SAME) {
        R::trim(wr, H, l);
        if (a.pw) R::trim(pwr, H, l);
        if (LAYER && a.pb) R::trim(pbr, H, l);
    }
    for (int64_t base = first; base < r1; base += stride) {    // (uniform in the workgroup)
        const bool valid = base + slot < r1;
        const int64_t row = row_at(base);
        const float live = valid ? 1.f : 0.f;
        const float mu = mean, rs = rstd, pmu = pmean, prs = prstd;
        float v[NE], n[NE], dr[NE], dy[NE], g[NE], p[NE];
        R::row(xr, H, l, v);
        if (a.h) R::row(hr, H, l, n);
        if (a.gate) R::row(gr, H, l, g);
        if (a.dy) R::row(dyr, H, l, dy);
        if (a.dr) R::row(drr, H, l, dr);
        else {
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = 0.f;
        }
        if (base + stride < r1) fetch(row_at(base + stride));
        auto pre_w = [&]() {
            if constexpr (SAME) R::expand(wr, p);
            else R::param(a.w, a.wdt, H, l, p);
        };
        auto post_w = [&]() {
            if constexpr (SAME) R::expand(pwr, p);
            else R::param(a.pw, a.wdt, H, l, p);
        };
        auto normed = [&](float (&t)[NE]) {                    // n of the forward: h, or post's result from n = hhat
#pragma unroll
            for (int e = 0; e < NE; ++e) t[e] = n[e];
            if (!a.pw) return;
            post_w();
#pragma unroll
            for (int e = 0; e < NE; ++e) t[e] *= p[e];
            if (LAYER && a.pb) {
                if constexpr (SAME) R::expand(pbr, p);
                else R::param(a.pb, a.wdt, H, l, p);
#pragma unroll
                for (int e = 0; e < NE; ++e) t[e] += p[e];
            }
        };
        if (a.h) {
            if (a.pw) {
#pragma unroll
                for (int e = 0; e < NE; ++e) n[e] = R::has(l, e, H) ? (n[e] - pmu) * prs : 0.f;
            }
            float t[NE];
            normed(t);
            if (a.gate) {
#pragma unroll
                for (int e = 0; e < NE; ++e) t[e] *= g[e];
            }
#pragma unroll
            for (int e = 0; e < NE; ++e) v[e] = fmaf(a.scale, t[e], v[e]);
        }
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = R::has(l, e, H) ? (v[e] - mu) * rs : 0.f;        // rhat
        if (a.dy) {
            float c1 = 0.f, c2 = 0.f;
            pre_w();
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                sw[e] = fmaf(live * dy[e], v[e], sw[e]);
                if constexpr (LAYER) sb[e] = fmaf(live, dy[e], sb[e]);
                dy[e] *= p[e];
                c1 = fmaf(dy[e], v[e], c1);
                if constexpr (LAYER) c2 += dy[e];
            }
            rn_sum<TPR, LAYER>(c1, c2, red, flip);
            c1 *= inv;
            c2 *= inv;
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = fmaf(rs, dy[e] - v[e] * c1 - c2, dr[e]);
        }
        if (valid) R::store(a.dx, row * H, H, l, dr);
        if (!a.h) continue;
#pragma unroll
        for (int e = 0; e < NE; ++e) dr[e] *= a.scale;
        if (a.gate) {
            float t[NE];
            normed(t);
#pragma unroll
            for (int e = 0; e < NE; ++e) t[e] *= dr[e];
            if (each) {
                if (valid) R::store(a.dgate, row * H, H, l, t);
            } else {
#pragma unroll
                for (int e = 0; e < NE; ++e) sg[e] = fmaf(live, t[e], sg[e]);
            }
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] *= g[e];                  // dn
        }
        if (a.pw) {
            float c1 = 0.f, c2 = 0.f;
            post_w();
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                if (!R::has(l, e, H)) dr[e] = 0.f;
                spw[e] = fmaf(live * dr[e], n[e], spw[e]);
                if constexpr (LAYER) spb[e] = fmaf(live, dr[e], spb[e]);
                dr[e] *= p[e];
                c1 = fmaf(dr[e], n[e], c1);
                if constexpr (LAYER) c2 += dr[e];
            }
            rn_sum<TPR, LAYER>(c1, c2, red, flip);
            c1 *= inv;
            c2 *= inv;
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = prs * (dr[e] - n[e] * c1 - c2);
        }
        if (a.dh && valid) R::store(a.dh, row * H, H, l, dr);
    }
    // sum over the workgroup's row slots -> put(column, sum)
    auto over_slots = [&](const float* s, auto put) {
        if constexpr (RB > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < NE; ++e) comb[(slot * NE + e) * TPR + l] = s[e];
            __syncthreads();
            if (slot == 0) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    float z = 0.f;
#pragma unroll
                    for (int k = 0; k < RB; ++k) z += comb[(k * NE + e) * TPR + l];
                    if (R::has(l, e, H)) put(R::col(l, e, H), z);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (R::has(l, e, H)) put(R::col(l, e, H), s[e]);
        }
    };
    float* out = a.part + (int64_t)blockIdx.x * a.narr * H;
    auto flush = [&](const float* s, int at) {
        if (at >= 0) over_slots(s, [&](int c, float z) { out[(int64_t)at * H + c] = a.add ? out[(int64_t)at * H + c] + z : z; });
    };
    flush(sw, a.s_w);
    if constexpr (LAYER) flush(sb, a.s_b);
    flush(spw, a.s_pw);
    if constexpr (LAYER) flush(spb, a.s_pb);
    if (a.gate && !each) {
        if (a.s_g >= 0) flush(sg, a.s_g);
        else over_slots(sg, [&](int c, float z) { store1<DT>(a.dgate, group * H + c, z); });      // the group's only workgroup
    }
}

struct RnSumArgs {
    const float* part;
    void* out[5];
    int dt[5];
    int64_t first[5], count[5], parts[5];   // slot, output rows, partial rows summed into each output row
    int n, H, narr;
};

// one output row (a parameter's gradient, or one row of a shared gate's) per blockIdx.y: 64 columns, 16 waves share the parts
__global__ __launch_bounds__(1024) void rn_sum_kernel(RnSumArgs a) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, H = a.H;
    const int nc = (H + 63) / 64, c = (int)(blockIdx.x % nc) * 64 + lane;
    int64_t o = blockIdx.x / nc;
    int k = 0;
    while (k < a.n - 1 && o >= a.count[k]) o -= a.count[k++];
    const int64_t parts = a.parts[k];
    const float* p = a.part + (o * parts * a.narr + a.first[k]) * H + c;
    float s = 0.f;
    if (c < H) {
#pragma unroll 8
        for (int64_t i = wave; i < parts; i += 16) s += p[i * a.narr * H];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < H) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += red[i][lane];
        if (a.dt[k] == DTF_BF16) store1<DTF_BF16>(a.out[k], o * H + c, s);
        else store1<DTF_F32>(a.out[k], o * H + c, s);
    }
}

// Threads of a row.  Forward 16 elements a thread.  Backward 8 (its sums and the next row's loads take the registers: 16 at
// width 4096 left two waves a SIMD, 250 us where 8 take 157), but no more than 512 threads to H = 8192: 1024 leave 128
// registers each, which spill (8192 rows of 8192, one norm: 145 against 139 us).
static int rn_tpr(int H, int ne) {
    if (H <= 512) return 64;
    if (H > 8192) return 1024;
    return H <= 64 * ne ? 64 : H <= 128 * ne ? 128 : H <= 256 * ne ? 256 : 512;
}

// Workgroups of the backward: nbx share a group's rows, gstep groups go into a launch.  8 waves a CU.  Backward and the sum
// of the parts behind it at 16384 rows, 8 against 16 waves a CU: width 4096 (rms, both norms) 157 + 6 against 164 + 9 us,
// 2048 105 + 5 / 119 + 8; layer norms at 768 (65536 rows) 162 + 5 / 156 + 8.
// More groups than a launch takes go one workgroup a group, launch after launch, and the last launch may be far from full: width
// 4096, both norms, 256 gate rows over 64 rows each 174 us, 257 288 (one workgroup walks 64 rows in a launch of its own); width
// 2048, 512 over 32 rows each 84, 513 142, 2048 over 8 each 125.
static void rn_grid(int64_t M, int H, int64_t groups, int* nbx, int64_t* gstep) {
    const int tpr = rn_tpr(H, 8), rb = tpr < 256 ? 256 / tpr : 1;
    const int64_t target = tpr <= 256 ? 512 : 256;
    const int64_t n = target / groups, most = ((M + groups - 1) / groups + rb - 1) / rb;
    *nbx = (int)(n < 1 ? 1 : n > most ? most : n);
    *gstep = groups < target ? groups : target;
}

extern "C" {

// What a call is about, packed by its caller (one pointer is cheaper to hand over than twenty arguments).  Rows [M, H]
// contiguous; gate [M / rpg, H] or null; w, b, pw, pb of type wdt (dt or fp32).
struct RnCall {
    int64_t M, rpg;
    int dt, wdt, layer, H;
    float scale, eps;
};
static_assert(sizeof(RnCall) == 40, "packed by the caller");

// fp32 workspace of the backward, in floats: groups = rows of a shared gate (1 without), narr = number of sums
int64_t dtf_residual_norm_ws(const RnCall* c, int64_t groups, int narr) {
    int nbx;
    int64_t gstep;
    rn_grid(c->M, c->H, groups, &nbx, &gstep);
    return gstep * nbx * narr * c->H;
}

#define RN_SHAPES_FWD(X, DTY, VECT)                                                               \
    if (H <= 512) { X(DTY, VECT, 64, 8) } else if (H <= 1024) { X(DTY, VECT, 64, 16) }            \
    else if (H <= 2048) { X(DTY, VECT, 128, 16) } else if (H <= 4096) { X(DTY, VECT, 256, 16) }   \
    else if (H <= 8192) { X(DTY, VECT, 512, 16) } else { X(DTY, VECT, 1024, 16) }
#define RN_SHAPES_BWD(X, DTY, VECT)                                                               \
    if (H <= 512) { X(DTY, VECT, 64, 8) } else if (H <= 1024) { X(DTY, VECT, 128, 8) }            \
    else if (H <= 2048) { X(DTY, VECT, 256, 8) } else if (H <= 4096) { X(DTY, VECT, 512, 8) }     \
    else if (H <= 8192) { X(DTY, VECT, 512, 16) } else { X(DTY, VECT, 1024, 16) }
#define RN_BY_TYPE(SHAPES, X, MODE)                                                              \
    if (dt == DTF_BF16) {                                                                        \
        if (H < 8) { X(DTF_BF16, RN_TINY, 64, 8) } else { SHAPES(X, DTF_BF16, MODE) }            \
    } else {                                                                                     \
        if (H < 4) { X(DTF_F32, RN_TINY, 64, 8) } else { SHAPES(X, DTF_F32, MODE) }              \
    }

static int rn_check(int dt, int wdt, int64_t M, int H, int64_t rpg) {
    if (dt != DTF_F32 && dt != DTF_BF16) return -90;
    if (wdt != dt && wdt != DTF_F32) return -90;
    if (M <= 0 || H <= 0 || H > 16384 || rpg <= 0) return -91;
    return 0;
}

// p: x, h, gate, w, b, pw, pb, y, r, stats (fp32 [4, M]); h and r, gate, b, pw, pb may be null
int dtf_residual_norm_fwd(void* const* p, const RnCall* c, hipStream_t stream) {
    DTF_CLEAR_ERRORS();
    const int dt = c->dt, H = c->H;
    const int64_t M = c->M;
    int rc = rn_check(dt, c->wdt, M, H, c->rpg);
    if (rc) return rc;
    RnArgs a{};
    a.x = p[0]; a.h = p[1]; a.gate = p[2]; a.w = p[3]; a.b = p[4]; a.pw = p[5]; a.pb = p[6]; a.y = p[7]; a.r = p[8]; a.stats = (float*)p[9];
    a.M = M; a.rpg = c->rpg; a.H = H; a.wdt = c->wdt; a.layer = c->layer; a.scale = c->scale; a.eps = c->eps;
    uintptr_t al = 0;
    for (int i = 0; i < 9; ++i) al |= (uintptr_t)p[i];
    const bool vec = !(al & 15) && H % (dt == DTF_BF16 ? 8 : 4) == 0;
    const int tpr = rn_tpr(H, 16), nt = tpr < 256 ? 256 : tpr, rb = nt / tpr;
    const int64_t grid = (M + rb - 1) / rb;
    if (grid > 0x7fffffff) return -92;
#define RN_FWD(DTY, VECT, TPR, NE) \
    hipLaunchKernelGGL((rn_fwd_kernel<DTY, VECT, TPR, NE>), dim3((unsigned)grid), dim3(nt), 0, stream, a);
    // (16384 rows of 2048: 45 us, 50 as rows that begin anywhere; the backward takes the same time either way)
    if (vec) { RN_BY_TYPE(RN_SHAPES_FWD, RN_FWD, RN_ALIGNED) } else { RN_BY_TYPE(RN_SHAPES_FWD, RN_FWD, RN_ANY) }
#undef RN_FWD
    DTF_CHECK_LAUNCH();
    return 0;
}

// p: x, h, gate, w, pw, pb, stats, dy, dr, dx, dh, dgate, dw, db, dpw, dpb, ws.  dgate [M, H] for a gate per element, else
// [M / rpg, H] through the partials; dw, db, dpw, dpb of type wdt; any of them null where there is no such operand.  ws:
// dtf_residual_norm_ws(c, groups, narr) floats, groups = M / rpg for a shared gate and 1 otherwise, narr = number of sums (dw,
// db, dpw, dpb, dgate of a shared gate) or more.
int dtf_residual_norm_bwd(void* const* p, const RnCall* c, hipStream_t stream) {
    DTF_CLEAR_ERRORS();
    const int dt = c->dt, wdt = c->wdt, layer = c->layer, H = c->H;
    const int64_t M = c->M, rpg = c->rpg;
    int rc = rn_check(dt, wdt, M, H, rpg);
    if (rc) return rc;
    void *h = p[1], *gate = p[2], *pw = p[4], *dgate = p[11], *dw = p[12], *db = p[13], *dpw = p[14], *dpb = p[15];
    float* ws = (float*)p[16];
    if (gate && (!dgate || !h)) return -93;
    RnArgs a{};
    a.x = p[0]; a.h = h; a.gate = gate; a.w = p[3]; a.pw = pw; a.pb = p[5]; a.stats = (float*)p[6]; a.dy = p[7]; a.dr = p[8];
    a.dx = p[9]; a.dh = p[10]; a.part = ws; a.M = M; a.rpg = rpg; a.H = H; a.wdt = wdt; a.layer = layer; a.scale = c->scale;
    const bool shared = gate && rpg > 1;
    a.dgate = dgate;
    const int64_t groups = shared ? (M + rpg - 1) / rpg : 1;
    a.group_rows = shared ? rpg : M;
    int64_t gstep;
    rn_grid(M, H, groups, &a.nbx, &gstep);
    RnSumArgs s{};
    auto sum = [&](void* out, int type, bool on, int64_t rows) {
        if (!on || !out) return -1;
        s.out[s.n] = out; s.dt[s.n] = type; s.first[s.n] = s.n; s.count[s.n] = rows;
        s.parts[s.n] = rows > 1 ? a.nbx : gstep * a.nbx;
        return s.n++;
    };
    a.s_w = sum(dw, wdt, true, 1);
    a.s_b = sum(db, wdt, layer, 1);
    a.s_pw = sum(dpw, wdt, pw != nullptr, 1);
    a.s_pb = sum(dpb, wdt, layer && pw, 1);
    a.s_g = sum(dgate, dt, shared && a.nbx > 1, groups);
    a.narr = s.n;
    const int tpr = rn_tpr(H, 8), nt = tpr < 256 ? 256 : tpr;
#define RN_BWD_L(DTY, VECT, TPR, NE, SM)                                                                                         \
    if (layer) hipLaunchKernelGGL((rn_bwd_kernel<DTY, VECT, TPR, NE, true, SM>), dim3((unsigned)grid), dim3(nt), 0, stream, a);  \
    else hipLaunchKernelGGL((rn_bwd_kernel<DTY, VECT, TPR, NE, false, SM>), dim3((unsigned)grid), dim3(nt), 0, stream, a);
#define RN_BWD(DTY, VECT, TPR, NE)                                                        \
    if (DTY == DTF_F32 || wdt == DTY) { RN_BWD_L(DTY, VECT, TPR, NE, true) }               \
    else { RN_BWD_L(DTY, VECT, TPR, NE, false) }
    for (; a.group0 < groups; a.group0 += gstep) {
        const int64_t grid = (groups - a.group0 < gstep ? groups - a.group0 : gstep) * a.nbx;
        a.add = a.group0 > 0;
        RN_BY_TYPE(RN_SHAPES_BWD, RN_BWD, RN_ANY)
        DTF_CHECK_LAUNCH();
    }
#undef RN_BWD
#undef RN_BWD_L
    if (s.n == 0) return 0;
    s.part = ws; s.H = H; s.narr = s.n;
    int64_t rows = 0;
    for (int i = 0; i < s.n; ++i) rows += s.count[i];
    rows *= (H + 63) / 64;
    if (rows > 0x7fffffff) return -92;
    hipLaunchKernelGGL(rn_sum_kernel, dim3((unsigned)rows), dim3(1024), 0, stream, s);
    DTF_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
