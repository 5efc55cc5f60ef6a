// K23: rotary positions (bf16 / fp32): pairs of a head's first 2m elements turn by the angle position * inv_freq[pair].
//
//   half        pair j = (x[j], x[j + m]);   interleaved: (x[2j], x[2j + 1]);   elements from 2m on pass through
//   y_a = A (x_a cos - x_b sin),  y_b = A (x_a sin + x_b cos);  backward: the same with sin negated
//
// The angle is position * inv_freq in 64 bits, reduced to a part of one turn there (a far position's angle has no
// fraction left in 32 bits), its sine and cosine in fp32.  A workgroup owns TB tokens: each of its threads computes one
// (token, pair)'s sine and cosine into LDS, then all heads of q and k of those tokens stream through it -- q and k are
// read and written once, no table of angles exists in memory.
// HBM-bound: 16384 tokens, 40 heads of 128, bf16: 335 MB in 63 us (5.3 TB/s), fp32 at half the tokens 57 us (5.9); 74 of the
// 128 turned 72 us (vectors that begin inside a dword).
#include "dtf_common.h"
#include <type_traits>

#define RO_PAIRS 1024          // (token, pair)s of a workgroup held in LDS
#define RO_UNROLL 4            // units in flight per thread

struct RoArgs {
    const void *q, *k;                                    // element (b, s, h, d) at b*bs + s*ss + h*hs + d
    void *qo, *ko;                                        // contiguous [B, S, H, D]
    int64_t q_bs, q_ss, q_hs, k_bs, k_ss, k_hs;
    const void* pos;                                      // int64 / int32 position of (b, s) at b*p_bs + s*p_ss; null: offset + s
    int64_t p_bs, p_ss, offset, tokens;                   // tokens = B * S
    const double* inv_freq;                               // [m]
    int S, Hq, Hk, D, m, tb, pos64;
    float amp, sign;
};

template <int V, int ESZ> struct RoVec;
template <> struct RoVec<8, 2> { typedef u32x4 type; };
template <> struct RoVec<4, 2> { typedef u32x2 type; };
template <> struct RoVec<2, 2> { typedef unsigned int type; };
template <> struct RoVec<4, 4> { typedef u32x4 type; };
template <> struct RoVec<2, 4> { typedef u32x2 type; };
template <> struct RoVec<1, 2> { typedef unsigned short type; };
template <> struct RoVec<1, 4> { typedef unsigned int type; };

template <int DT, int V>
__device__ __forceinline__ void ro_unpack(const typename RoVec<V, DT == DTF_BF16 ? 2 : 4>::type& r, float (&x)[V]) {
    if constexpr (V == 1) {
        if constexpr (DT == DTF_BF16) x[0] = bf16_to_f32(r);
        else x[0] = __uint_as_float(r);
    } else {
        unsigned int w[DT == DTF_BF16 ? V / 2 : V];
        __builtin_memcpy(w, &r, sizeof(w));
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if constexpr (DT == DTF_BF16) x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
            else x[e] = __uint_as_float(w[e]);
        }
    }
}

template <int DT, int V>
__device__ __forceinline__ typename RoVec<V, DT == DTF_BF16 ? 2 : 4>::type ro_pack(const float (&x)[V]) {
    typename RoVec<V, DT == DTF_BF16 ? 2 : 4>::type r;
    if constexpr (V == 1) {
        if constexpr (DT == DTF_BF16) r = f32_to_bf16(x[0]);
        else r = __float_as_uint(x[0]);
    } else {
        unsigned int w[DT == DTF_BF16 ? V / 2 : V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if constexpr (DT == DTF_F32) w[e] = __float_as_uint(x[e]);
            else if (e & 1) w[e / 2] = pack_bf16x2(x[e - 1], x[e]);
        }
        __builtin_memcpy(&r, w, sizeof(w));
    }
    return r;
}

// A unit is V pairs (two vectors of V elements) or, past 2m, two vectors that pass through.  A last unit that would pass the
// end of its range lies over the one before it (both write the same values); less than a vector past 2m is stored by words.
// Vectors begin anywhere: the hardware takes them unaligned.
template <int DT, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RoArgs a) {
    constexpr int ESZ = DT == DTF_BF16 ? 2 : 4;
    typedef typename RoVec<V, ESZ>::type vec __attribute__((aligned(ESZ)));
    typedef typename std::conditional<DT == DTF_BF16, unsigned short, unsigned int>::type elem;
    typedef unsigned int word __attribute__((aligned(2)));
    __shared__ __attribute__((aligned(16))) float cs[RO_PAIRS], sn[RO_PAIRS];
    const int tid = threadIdx.x, m = a.m;
    const int64_t t0 = (int64_t)blockIdx.x * a.tb;
    const int nt = (int)(a.tokens - t0 < a.tb ? a.tokens - t0 : a.tb);
    for (int p = tid; p < nt * m; p += 256) {
        const int tt = p / m, j = p - tt * m;
        const int64_t t = t0 + tt, b = t / a.S, s = t - b * a.S;
        int64_t pos = a.offset + s;
        if (a.pos) {
            const int64_t at = b * a.p_bs + s * a.p_ss;
            pos = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at] : (int64_t) reinterpret_cast<const int*>(a.pos)[at];
        }
        const double turns = (double)pos * a.inv_freq[j] * 0.15915494309189533577;      // 1 / (2 pi)
        float sv, cv;
        sincospif((float)(2.0 * (turns - rint(turns))), &sv, &cv);
        cs[p] = cv * a.amp;
        sn[p] = sv * a.amp * a.sign;
    }
    __syncthreads();
    const int rest = a.D - 2 * m, rot = (m + V - 1) / V, U = rot + (rest + 2 * V - 1) / (2 * V), H = a.Hq + a.Hk, total = nt * H * U;
    for (int i0 = tid; i0 < total; i0 += 256 * RO_UNROLL) {
        vec x[RO_UNROLL], y[RO_UNROLL];
        elem* dst[RO_UNROLL];
        int pr[RO_UNROLL], dist[RO_UNROLL];
#pragma unroll
        for (int n = 0; n < RO_UNROLL; ++n) {
            const int i = min(i0 + n * 256, total - 1);                   // past the end: the last unit again, not stored
            const int w = i / U, u = i - w * U, tt = w / H, h = w - tt * H;
            const int64_t t = t0 + tt, b = t / a.S, s = t - b * a.S;
            const bool is_q = h < a.Hq;
            const elem* src = is_q ? (const elem*)a.q + b * a.q_bs + s * a.q_ss + h * a.q_hs
                                   : (const elem*)a.k + b * a.k_bs + s * a.k_ss + (h - a.Hq) * a.k_hs;
            dst[n] = is_q ? (elem*)a.qo + (t * a.Hq + h) * a.D : (elem*)a.ko + (t * a.Hk + (h - a.Hq)) * a.D;
            const bool turn = u < rot;
            const int j = min(u * V, m - V);                              // a turning unit's first pair
            const int first = turn ? (INTER ? 2 * j : j) : 2 * m + min((u - rot) * 2 * V, rest < V ? rest - V : max(0, rest - 2 * V));
            dist[n] = turn ? (INTER ? V : m) : max(0, min(V, rest - V));
            pr[n] = turn ? tt * m + j : -1;
            dst[n] += first;
            x[n] = *reinterpret_cast<const vec*>(src + first);
            y[n] = *reinterpret_cast<const vec*>(src + first + dist[n]);
        }
#pragma unroll
        for (int n = 0; n < RO_UNROLL; ++n) {
            if (i0 + n * 256 >= total) break;
            if (pr[n] >= 0) {
                float p[V], q[V];
                ro_unpack<DT, V>(x[n], p);
                ro_unpack<DT, V>(y[n], q);
                if constexpr (INTER) {                                    // 2V consecutive elements hold V pairs
                    float z[2 * V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        z[e] = p[e];
                        z[V + e] = q[e];
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float c = cs[pr[n] + e], s = sn[pr[n] + e], xa = z[2 * e], xb = z[2 * e + 1];
                        z[2 * e] = xa * c - xb * s;
                        z[2 * e + 1] = xa * s + xb * c;
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        p[e] = z[e];
                        q[e] = z[V + e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float c = cs[pr[n] + e], s = sn[pr[n] + e], xa = p[e], xb = q[e];
                        p[e] = xa * c - xb * s;
                        q[e] = xa * s + xb * c;
                    }
                }
                x[n] = ro_pack<DT, V>(p);
                y[n] = ro_pack<DT, V>(q);
            } else if (rest < V) {
                if constexpr (V * ESZ > 4) {                              // (V > 2: rest is even)
#pragma unroll
                    for (int k = 0; k < V * ESZ / 4; ++k)
                        if (k * 4 >= (V - rest) * ESZ) reinterpret_cast<word*>(dst[n])[k] = x[n][k];
                }
                continue;
            }
            *reinterpret_cast<vec*>(dst[n]) = x[n];
            *reinterpret_cast<vec*>(dst[n] + dist[n]) = y[n];
        }
    }
}

extern "C" {

// A call, packed by its caller (one pointer is cheaper to hand over than twenty arguments).  k and ko may be null (Hk = 0).
// pos: null, or int32 / int64 (pos64) with strides p_bs, p_ss.  st: element strides (batch, token, head) of q, then of k.
// sign: +1 forward, -1 backward.
struct RoCall {
    const void *q, *k;
    void *qo, *ko;
    const void* pos;
    const double* inv_freq;
    int64_t st[6], p_bs, p_ss, offset;
    int dt, pos64, B, S, Hq, Hk, D, m, interleaved;
    float amp, sign;
    int pad;
};
static_assert(sizeof(RoCall) == 168, "packed by the caller");

int dtf_rotary(const RoCall* c, hipStream_t stream) {
    DTF_CLEAR_ERRORS();
    const int dt = c->dt, B = c->B, S = c->S, Hq = c->Hq, Hk = c->Hk, D = c->D, m = c->m, interleaved = c->interleaved;
    if (B <= 0 || S <= 0 || Hq <= 0 || Hk < 0 || D <= 0 || m <= 0 || 2 * m > D || m > RO_PAIRS || (D & 1)) return -80;
    if (dt != DTF_F32 && dt != DTF_BF16) return -81;
    RoArgs a{c->q, c->k, c->qo, c->ko, c->st[0], c->st[1], c->st[2], c->st[3], c->st[4], c->st[5], c->pos, c->p_bs, c->p_ss,
             c->offset, (int64_t)B * S, c->inv_freq, S, Hq, Hk, D, m, 1, c->pos64, c->amp, c->sign};
    // elements a load: 16 B, or the largest half that fits the pairs (16384 tokens, 40 heads, 76 of 128 turned, bf16: 66 us; by
    // 8 B 85, by 4 B 130)
    int V = dt == DTF_BF16 ? 8 : 4;
    while (m < V) V >>= 1;
    // tokens of a workgroup: about RO_UNROLL units a thread (34440 tokens with 2 heads of 96, fp32: 32 us, 42 with one unit each)
    const int64_t units = (int64_t)(Hq + Hk) * ((m + V - 1) / V + (D - 2 * m + 2 * V - 1) / (2 * V));
    if (units > 0x40000000) return -82;
    int tb = (int)(256 * RO_UNROLL / units);
    if (tb > RO_PAIRS / m) tb = RO_PAIRS / m;
    if (tb < 1) tb = 1;
    a.tb = tb;
    const int64_t grid = (a.tokens + tb - 1) / tb;
    if (grid > 0x7fffffff) return -82;
#define RO_LAUNCH(DTY, VV)                                                                                               \
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<DTY, VV, true>), dim3((unsigned)grid), dim3(256), 0, stream, a);  \
    else hipLaunchKernelGGL((rotary_kernel<DTY, VV, false>), dim3((unsigned)grid), dim3(256), 0, stream, a);
    if (dt == DTF_BF16) {
        if (V == 8) { RO_LAUNCH(DTF_BF16, 8) } else if (V == 4) { RO_LAUNCH(DTF_BF16, 4) }
        else if (V == 2) { RO_LAUNCH(DTF_BF16, 2) } else { RO_LAUNCH(DTF_BF16, 1) }
    } else {
        if (V == 4) { RO_LAUNCH(DTF_F32, 4) } else if (V == 2) { RO_LAUNCH(DTF_F32, 2) } else { RO_LAUNCH(DTF_F32, 1) }
    }
#undef RO_LAUNCH
    DTF_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
