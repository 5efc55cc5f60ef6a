// K22: attention of any length on gfx950 -- bf16, head dims to 128, grouped heads, causal or with key lengths, strided
// operands; forward and the backward that recomputes the probabilities.
//
//   vis(i) = number of keys that query i sees (always a prefix): min(kv_len[b], causal ? i + 1 + Sk - Sq : Sk), >= 0
//   S = c Q K^T,  P = softmax over the vis(i) keys (no key: P = 0),  O = P V
//   D = rowsum(dO o O),  dP = dO V^T,  dS = P o (dP - D),  dQ = c dS K,  dK = c dS^T Q,  dV = P^T dO
//
// One online-softmax pass over the keys, 32x32x16 MFMA tiles:
//   S^T = K . Q^T      a lane owns ONE query (column lane & 31) and 16 of a tile's 32 keys, so the running maximum and
//                      sum are register reductions plus one exchange with lane ^ 32
//   O^T = V^T . P^T    the score accumulator, rounded to bf16, IS the B operand: registers 8s .. 8s+7 of a lane hold the
//                      keys 16s + 8 (j >> 2) + 4 g + (j & 3), j = 0..7, g = lane >> 5; the A operand V^T comes in that
//                      key order from two ds_read_b64_tr_b16
// Bound by the matrix pipe and by power: 4 x 4096 tokens, 16 heads of 128, not causal: forward 555 us (990 TF/s), dQ 757 us
// (1090 in its three products), dK/dV 1060 us (1040 in its four), where a large library product makes 1400..1600; the card
// lowers its clock under them (1.8 of 2.4 GHz; on zeros instead of random values the same kernels take a fifth less).
// Two waves a SIMD carry it (heads to 64: four in the forward, three in the backward): with 64 queries a wave (half the LDS
// reads, one wave a SIMD) the forward took 918 us, with 32-key steps (three waves) 556, the next step's scores issued under this
// one's exponentials 640.  LDS reads are one operand of every product, 33..46 % of its cycles.
// P and dS are rounded to bf16 for the second products (their operands' type: off by half a step, up to 2^-8 of each term and
// 1.65e-3 of it in the mean square, random in sign, so the sums keep the accuracy of the bf16 results, whose own rounding is as
// large: 2.4e-3 of the norm in all); scores, maxima, sums, L, D and all accumulators are fp32.
#include "dtf_common.h"

typedef __attribute__((ext_vector_type(4))) short ag_s16x4;
typedef __attribute__((address_space(3))) void ag_lds_void;
typedef unsigned short u16;

#define AG_NEG (-__builtin_inff())

struct AgArgs {
    const u16 *q, *k, *v;                 // element (b, s, h, d) of T at T + b*T_bs + s*T_ss + h*T_hs + d
    int64_t q_bs, q_ss, q_hs, k_bs, k_ss, k_hs, v_bs, v_ss, v_hs;
    const u16 *o, *dO;                    // contiguous [B, Sq, Hq, D]
    u16 *out, *dq, *dk, *dv;              // contiguous [B, Sq, Hq, D] (dk, dv: [B, Sk, Hk, D])
    float *lse, *dsum;                    // [B, Hq, Sq]; lse in the log2 domain, +inf for a query that sees no key
    const int* kv_len;                    // [B] or null
    float* ws;                            // partial results of `nsplit` workgroups that share a tile; unused for nsplit = 1
    int B, Sq, Sk, Hq, Hk, D, group, causal, ntiles, nsplit;
    float scale, scale_log2e;
};

// Tiles are DP = 64 or 128 columns wide in LDS, of which loads and products take DC = 32, 64, 96 or 128 (D, rounded up to 32).
// Against DC = DP, 4 x 4096 tokens, 8 heads of 32: forward 162 -> 139 us, backward 558 -> 380; of 96: 270 -> 240, 865 -> 757.
// LDS image of a [rows][DP] bf16 tile, 16-B chunk c of row r, without bank conflicts (256 B of banks) for ds_read_b128 of 16
// rows at one chunk and for ds_read_b64_tr_b16 of 4 rows x 32 columns: the 32-B chunk is XORed so that rows 0..3 of a
// 4-row block take different PAIRS of chunks (a plain XOR with the row puts rows 0 and 1 on the same pair: 2 extra cycles
// a transposed read, a quarter of the LDS time), rows + 4 the odd places, rows + 8 the other 16-B half.
template <int DP>
__device__ __forceinline__ int ag_swz(int row) {
    return DP == 128 ? (row & 3) << 1 | ((row >> 2) & 1) : (row & 2) | ((row >> 2) & 1);
}
template <int DP>
__device__ __forceinline__ int ag_off(int row, int c) {
    return row * (2 * DP) + ((((c >> 1) ^ ag_swz<DP>(row)) << 5) | (((c ^ (row >> 3)) & 1) << 4));
}

__device__ __forceinline__ f32x16 ag_zero() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

__device__ __forceinline__ f32x16 ag_mfma(s16x8 a, s16x8 b, f32x16 c) {
    typedef __attribute__((ext_vector_type(8))) __bf16 bf8;
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

// registers 8s .. 8s+7 of an accumulator as a bf16 operand
__device__ __forceinline__ s16x8 ag_pack(const f32x16& x, int s) {
    const u32x4 p = {pack_bf16x2(x[8 * s], x[8 * s + 1]), pack_bf16x2(x[8 * s + 2], x[8 * s + 3]),
                     pack_bf16x2(x[8 * s + 4], x[8 * s + 5]), pack_bf16x2(x[8 * s + 6], x[8 * s + 7])};
    return __builtin_bit_cast(s16x8, p);
}

// A lane's places in an image.  The swizzle is an XOR, so every other place is (place ^ constant) + constant:
//   row:   chunk g of row lane & 31; the k-th operand of 16 columns is at row ^ (k << 5), 32 rows further + 32 rows
//   tr:    the transposed read of rows 4 g + (0..3), columns 0..31 (the 16 lanes of a group read a 4-row x 16-column block,
//          lane 4 q + p its row q, columns 4 p); columns 32 d .. at tr ^ (d << 6), rows + 8 at (tr ^ 16) + 8 rows
// keep() makes the compiler derive them where they are used instead of holding 24 addresses over the loop (which spilled).
template <int DP>
struct AgLane {
    unsigned row, tr;
    __device__ __forceinline__ void init(int lane) {
        row = ag_off<DP>(lane & 31, lane >> 5);
        const int r = 4 * (lane >> 5) + ((lane >> 2) & 3), c = (lane & 16) + 4 * (lane & 3);
        tr = ag_off<DP>(r, c >> 3) + (c & 7) * 2;
    }
    __device__ __forceinline__ void keep() { asm volatile("" : "+v"(row), "+v"(tr)); }
    // rows r0 + (lane & 31) (r0 a multiple of 32), columns 16 k + 8 g .. + 7
    __device__ __forceinline__ s16x8 rows(const unsigned char* img, int r0, int k) const {
        return *reinterpret_cast<const s16x8*>(img + (row ^ (unsigned)(k << 5)) + r0 * DP * 2);
    }
    // transposed: columns 32 d .. + 31 as rows, image rows r0 .. r0 + 15 (r0 a multiple of 16) as k in the accumulators' order
    __device__ __forceinline__ s16x8 cols(const unsigned char* img, int r0, int d) const {
        typedef __attribute__((address_space(3))) ag_s16x4* lp;
        const ag_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(img + (tr ^ (unsigned)(d << 6)) + r0 * DP * 2));
        const ag_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(img + (tr ^ (unsigned)(d << 6 | 16)) + (r0 + 8) * DP * 2));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// A tile of ROWS rows from memory to an image by LDS-DMA (global_load_lds, 16 B a lane: no staging registers, no ds_write
// pass).  One wave instruction fills 1 KB = 1024 / (2 DP) image rows, so the chunk that a lane fetches is the one whose
// swizzled place it fills.  Rows at or past `limit` and columns past D come from a page of zeros: whatever padding holds is
// never read, and nothing masked reaches a product.
__device__ const u32x4 ag_zeros = {0u, 0u, 0u, 0u};
__device__ const float ag_inf = __builtin_inff();
typedef __attribute__((address_space(1))) const void ag_glb_void;

template <int DP, int DC, int ROWS, int NT>
struct AgTile {
    static constexpr int RPI = 1024 / (2 * DP), N = ROWS / RPI / (NT / 64), STEP = RPI * (NT / 64);
    const char* base;        // of the matrix (uniform)
    int64_t rs;              // bytes from row to row
    unsigned off;            // this lane's byte offset from the tile's first row (a token stride is below 2^25 elements)
    int row, c;              // this lane's tile row and chunk
    __device__ __forceinline__ void init(const u16* base_, int64_t rs_, int wave, int lane) {
        row = wave * RPI + lane / (DP / 8);
        const int p = lane % (DP / 8);
        // (STEP is a multiple of 16: the same chunk for every row of a lane)
        c = (((p >> 1) ^ ag_swz<DP>(row)) << 1) | ((p ^ (row >> 3)) & 1);
        base = reinterpret_cast<const char*>(base_);
        rs = rs_ * 2;
        off = (unsigned)row * (unsigned)rs + c * 16;
    }
    // rows row0 .. row0 + ROWS - 1 of the matrix; columns past DC stay as they are (nothing reads them)
    __device__ __forceinline__ void load(unsigned char* img, int row0, int limit, int D, int wave) const {
        const bool full = D == DC && row0 + ROWS <= limit;                 // (uniform)
        if (DC < DP && c * 8 >= DC) return;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const char* p = base + (row0 + i * STEP) * rs;
            const void* from = p + off;
            if (!full && !(c * 8 < D && row0 + row + i * STEP < limit)) from = &ag_zeros;
            __builtin_amdgcn_global_load_lds((ag_glb_void*)from, (ag_lds_void*)(img + (i * (NT / 64) + wave) * 1024), 16, 0, 0);
        }
    }
};

// Workgroup order: the tile is the slow index (causal tiles differ in length: all heads' longest come first, and every XCD
// gets the same mix), the unit -- (share, head) -- the fast one.  Ids go round the 8 XCDs, so with a multiple of 8 units one
// head's workgroups stay on one XCD and its keys and values in one L2; so do the query heads of one key head.
__device__ __forceinline__ int ag_vis(const AgArgs& a, int i, int klen) {
    int n = a.causal ? min(klen, i + 1 + a.Sk - a.Sq) : klen;
    return max(n, 0);
}

__device__ __forceinline__ int ag_klen(const AgArgs& a, int b) { return a.kv_len ? max(0, min(a.kv_len[b], a.Sk)) : a.Sk; }

template <int DC>
__device__ __forceinline__ void ag_frags(s16x8 (&f)[DC / 16], const u16* row, int g, int D) {
#pragma unroll
    for (int ks = 0; ks < DC / 16; ++ks) {
        f[ks] = (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
        if (16 * ks + 8 * g < D) f[ks] = *reinterpret_cast<const s16x8*>(row + 16 * ks + 8 * g);
    }
}

// accumulator tiles [32 d][this lane's row] -> 4 bf16 at a time
template <int DC>
__device__ __forceinline__ void ag_store_row(u16* row, const f32x16 (&acc)[DC / 32], float f, int g, int D) {
#pragma unroll
    for (int dt = 0; dt < DC / 32; ++dt)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
            const int d = 32 * dt + 8 * rq + 4 * g;
            if (32 * dt + 8 * rq < D) {                                     // (uniform: D is a multiple of 8)
                const u32x2 p = {pack_bf16x2(acc[dt][4 * rq] * f, acc[dt][4 * rq + 1] * f),
                                 pack_bf16x2(acc[dt][4 * rq + 2] * f, acc[dt][4 * rq + 3] * f)};
                *reinterpret_cast<u32x2*>(row + d) = p;
            }
        }
}

// the same as fp32 sums
template <int DC>
__device__ __forceinline__ void ag_store_part(float* row, const f32x16 (&acc)[DC / 32], int g, int D) {
#pragma unroll
    for (int dt = 0; dt < DC / 32; ++dt)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
            if (32 * dt + 8 * rq < D)
                *reinterpret_cast<f32x4*>(row + 32 * dt + 8 * rq + 4 * g) =
                    (f32x4){acc[dt][4 * rq], acc[dt][4 * rq + 1], acc[dt][4 * rq + 2], acc[dt][4 * rq + 3]};
}

#define AG_LANDED() asm volatile("s_waitcnt vmcnt(0)" ::: "memory")      // this wave's LDS-DMA has arrived

// ---------------------------------------------------------------------------
// Forward: 4 waves x 32 queries, 64 keys a step, K and V double-buffered (the DMA of a step's successor runs under its
// products; one barrier a step).  The running maximum moves, and O is rescaled, only when a query's scores pass it by 2^8.
// PACK: the rows of a workgroup run over the `group` query heads of one key head and their Sq queries, so a few queries with
// many heads still fill the matrix tile and read K, V once.  nsplit > 1: that many workgroups share a tile's keys, each
// writes its (O, m, l), and ag_join_kernel adds them.
// ---------------------------------------------------------------------------
template <int DP, int DC, bool PACK>
__global__ __launch_bounds__(256, 2) void ag_fwd_kernel(AgArgs a) {
    constexpr int KS = DC / 16, DT = DC / 32, BN = 64, BM = 128;
    __shared__ __attribute__((aligned(16))) unsigned char K0[BN * DP * 2], K1[BN * DP * 2], V0[BN * DP * 2], V1[BN * DP * 2];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = a.B * a.Hk, units = gridDim.x / a.ntiles;               // units: nsplit x (PACK ? 1 : group) x kv
    const int t = a.ntiles - 1 - blockIdx.x / units, u = blockIdx.x % units;
    const int b = u % kv / a.Hk, hk = u % kv % a.Hk;
    const int h = PACK ? hk : hk * a.group + u / kv % a.group, sp = PACK ? u / kv : u / kv / a.group;
    const int rows = PACK ? a.group * a.Sq : a.Sq;
    const int klen = ag_klen(a, b);
    const int rw = t * BM + wave * 32, r = min(rw + (lane & 31), rows - 1);
    const int i = PACK ? r % a.Sq : r, head = PACK ? h * a.group + r / a.Sq : h;
    const int vis = ag_vis(a, i, klen);
    const int r0 = t * BM, r1 = min(t * BM + BM, rows) - 1;
    const int end = ag_vis(a, PACK ? (r0 / a.Sq == r1 / a.Sq ? r1 % a.Sq : a.Sq - 1) : r1, klen);
    int lo = vis, hi = rw < rows ? vis : 0;                                // of this wave's queries
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int steps = (end + BN - 1) / BN;
    const int kbeg = (int)((int64_t)steps * sp / a.nsplit) * BN, kend = min((int)((int64_t)steps * (sp + 1) / a.nsplit) * BN, end);

    s16x8 qf[KS];
    ag_frags<DC>(qf, a.q + b * a.q_bs + i * a.q_ss + head * a.q_hs, g, a.D);
    AgTile<DP, DC, BN, 256> kt, vt;
    kt.init(a.k + b * a.k_bs + hk * a.k_hs, a.k_ss, wave, lane);
    vt.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ss, wave, lane);
    auto fetch = [&](unsigned char* K, unsigned char* V, int k0) {
        kt.load(K, k0, klen, a.D, wave);
        vt.load(V, k0, klen, a.D, wave);
    };

    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = ag_zero();
    float m = AG_NEG, l = 0.f;
    AgLane<DP> at;
    at.init(lane);
    auto step = [&](const unsigned char* K, const unsigned char* V, int k0) {
        at.keep();
        f32x16 s[BN / 32];
#pragma unroll
        for (int u = 0; u < BN / 32; ++u) s[u] = ag_zero();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) s[u] = ag_mfma(at.rows(K, 32 * u, ks), qf[ks], s[u]);
        // reads run PF ahead of their products (left alone, the compiler waits for two at a time)
        constexpr int NR = KS * (BN / 32), PF = NR < 8 ? NR : 8;
        __builtin_amdgcn_sched_group_barrier(0x100, PF, 0);
#pragma unroll
        for (int z = 0; z < NR - PF; ++z) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, PF, 0);
        // a wave past its scores goes first: the SIMD's other wave has products to issue meanwhile (decoder 363 -> 329 us)
        __builtin_amdgcn_s_setprio(1);
        if (k0 + BN > lo) {
            const int left = vis - (k0 + 4 * g);
#pragma unroll
            for (int u = 0; u < BN / 32; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[u][e] = 32 * u + 8 * (e >> 2) + (e & 3) < left ? s[u][e] : AG_NEG;
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < BN / 32; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, s[u][e]);
        mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2e;
        // (a query's own affair: its bits do not depend on the wave's other queries)
        const bool up = !(mx <= m + 8.f);
        if (__any(up)) {
            const float mn = up ? __builtin_elementwise_maximum(m, mx) : m;
            const float alpha = mn == AG_NEG ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[dt][e] *= alpha;
        }
        const float mu = m == AG_NEG ? 0.f : m;                            // nothing seen yet: every p is exp2(-inf) = 0
#pragma unroll
        for (int u = 0; u < BN / 32; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], a.scale_log2e, -mu));
                l += s[u][e];
            }
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                const s16x8 pf = ag_pack(s[u], h2);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) oacc[dt] = ag_mfma(at.cols(V, 32 * u + 16 * h2, dt), pf, oacc[dt]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };
    if (kbeg < kend) fetch(K0, V0, kbeg);
    AG_LANDED();
    __syncthreads();
    for (int k0 = kbeg; k0 < kend; k0 += 2 * BN) {
        if (k0 + BN < kend) fetch(K1, V1, k0 + BN);
        if (k0 < hi) step(K0, V0, k0);
        AG_LANDED();
        __syncthreads();
        if (k0 + BN >= kend) break;
        if (k0 + 2 * BN < kend) fetch(K0, V0, k0 + 2 * BN);
        if (k0 + BN < hi) step(K1, V1, k0 + BN);
        AG_LANDED();
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    if (rw + (lane & 31) >= rows) return;
    const int64_t row = ((int64_t)b * a.Sq + i) * a.Hq + head;
    if (a.nsplit == 1) {
        ag_store_row<DC>(a.out + row * a.D, oacc, l == 0.f ? 0.f : 1.f / l, g, a.D);
        if (g == 0) a.lse[((int64_t)b * a.Hq + head) * a.Sq + i] = l == 0.f ? __builtin_inff() : m + log2f(l);
        return;
    }
    const int64_t n = (int64_t)a.B * a.Sq * a.Hq;
    ag_store_part<DC>(a.ws + (sp * n + row) * a.D, oacc, g, a.D);
    if (g == 0) {
        float* ml = a.ws + (int64_t)a.nsplit * n * a.D + (sp * n + row) * 2;
        ml[0] = m;
        ml[1] = l;
    }
}

// O = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).  A row: 32 lanes of 4 columns x PY threads that share the parts (few rows
// have many parts, and a chain of dependent reads per part cost more than the attention before it); 8 / PY rows a workgroup.
template <int PY>
__global__ __launch_bounds__(256) void ag_join_kernel(AgArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 os[8][32];
    __shared__ float ms[8], ls[8];
    const int x = threadIdx.x % 32, z = threadIdx.x / 32, y = z % PY, d = x * 4;
    const int64_t n = (int64_t)a.B * a.Sq * a.Hq, want = (int64_t)blockIdx.x * (8 / PY) + z / PY, row = want < n ? want : n - 1;
    const float* ml = a.ws + (int64_t)a.nsplit * n * a.D + row * 2;
    float m = AG_NEG, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = y; s < a.nsplit; s += PY) m = __builtin_elementwise_maximum(m, ml[s * n * 2]);
    for (int s = y; s < a.nsplit; s += PY) {
        const float mp = ml[s * n * 2], w = mp == AG_NEG ? 0.f : __builtin_amdgcn_exp2f(mp - m);
        l = fmaf(ml[s * n * 2 + 1], w, l);
        if (d < a.D) {
            const f32x4 p = *reinterpret_cast<const f32x4*>(a.ws + (s * n + row) * a.D + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(p[e], w, o[e]);
        }
    }
    os[z][x] = o;
    if (x == 0) {
        ms[z] = m;
        ls[z] = l;
    }
    __syncthreads();
    if (y > 0 || want >= n) return;
#pragma unroll
    for (int k = 1; k < PY; ++k) m = __builtin_elementwise_maximum(m, ms[z + k]);
    l = 0.f;
    o = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < PY; ++k) {
        const float w = ms[z + k] == AG_NEG ? 0.f : __builtin_amdgcn_exp2f(ms[z + k] - m);
        l = fmaf(ls[z + k], w, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(os[z + k][x][e], w, o[e]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d < a.D) {
        const u32x2 p = {pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2*>(a.out + row * a.D + d) = p;
    }
    if (x == 0) {
        const int64_t b = row / ((int64_t)a.Sq * a.Hq), ih = row - b * a.Sq * a.Hq, i = ih / a.Hq, h = ih - i * a.Hq;
        a.lse[(b * a.Hq + h) * a.Sq + i] = l == 0.f ? __builtin_inff() : m + log2f(l);
    }
}

// ---------------------------------------------------------------------------
// Backward, dQ: 4 waves x 32 queries, 64 keys a step.  nsplit > 1: as in the forward, that many workgroups share a tile's
// keys; they write fp32 sums.
// D = rowsum(dO o O) comes from the rounded O, whose half step weighs most where a query sees few keys (dS is then a
// difference of like terms: 16 tokens, causal: error of dq against 64 bits 3.0e-3 of its norm, 256 tokens 2.6e-3, where one
// rounding of the result makes 1.65e-3).  Tiles that see up to AG_FEW keys therefore sweep their keys twice and take
// D = sum P dP in fp32 first: 2.4e-3 at every length (8 x 512 tokens with AG_FEW 512: 31 us, with 256: 22 us, as exact).
// A query with ONE key has O = that V row: its D is the diagonal of O . dO^T by the matrix instruction, summed over d in the
// order of dP = V . dO^T, so its dS is 0 exactly.
// ---------------------------------------------------------------------------
#define AG_FEW 256

template <int DP, int DC>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void ag_dq_kernel(AgArgs a) {
    constexpr int KS = DC / 16, DT = DC / 32, BN = 64, BM = 128;
    __shared__ __attribute__((aligned(16))) unsigned char K0[BN * DP * 2], K1[BN * DP * 2], V0[BN * DP * 2], V1[BN * DP * 2];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = a.B * a.Hk, units = gridDim.x / a.ntiles;               // units: nsplit x group x kv
    const int t = a.ntiles - 1 - blockIdx.x / units, u = blockIdx.x % units;
    const int b = u % kv / a.Hk, hk = u % kv % a.Hk, h = hk * a.group + u / kv % a.group;
    const int sp = u / kv / a.group;
    const int klen = ag_klen(a, b);
    const int rw = t * BM + wave * 32, i = min(rw + (lane & 31), a.Sq - 1);
    const int vis = ag_vis(a, i, klen), end = ag_vis(a, min(t * BM + BM, a.Sq) - 1, klen);
    const int lo = ag_vis(a, min(rw, a.Sq - 1), klen), hi = rw < a.Sq ? ag_vis(a, min(rw + 32, a.Sq) - 1, klen) : 0;

    const int64_t row = ((int64_t)b * a.Sq + i) * a.Hq + h, li = ((int64_t)b * a.Hq + h) * a.Sq + i;
    s16x8 qf[KS], gf[KS];
    ag_frags<DC>(qf, a.q + b * a.q_bs + i * a.q_ss + h * a.q_hs, g, a.D);
    ag_frags<DC>(gf, a.dO + row * a.D, g, a.D);
    AgTile<DP, DC, BN, 256> kt, vt;
    kt.init(a.k + b * a.k_bs + hk * a.k_hs, a.k_ss, wave, lane);
    vt.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ss, wave, lane);
    auto fetch = [&](unsigned char* K, unsigned char* V, int k0) {
        kt.load(K, k0, klen, a.D, wave);
        vt.load(V, k0, klen, a.D, wave);
    };
    const int steps = (end + BN - 1) / BN;
    const int kbeg = (int)((int64_t)steps * sp / a.nsplit) * BN, kend = min((int)((int64_t)steps * (sp + 1) / a.nsplit) * BN, end);
    float dsum = 0.f;
    {
        s16x8 of[KS];
        ag_frags<DC>(of, a.o + row * a.D, g, a.D);
        f32x16 x = ag_zero();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x = ag_mfma(of[ks], gf[ks], x);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (8 * (e >> 2) + 4 * g + (e & 3) == (lane & 31)) dsum = x[e];
        dsum += __shfl_xor(dsum, 32, 64);
    }
    const float lse = a.lse[li];
    const bool valid = rw + (lane & 31) < a.Sq;

    AgLane<DP> at;
    at.init(lane);
    // scores (not seen: -inf) and dP of 32 keys
    auto products = [&](const unsigned char* K, const unsigned char* V, int k0, int u, f32x16& s, f32x16& dp) {
        s = ag_zero();
        dp = ag_zero();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s = ag_mfma(at.rows(K, 32 * u, ks), qf[ks], s);
            dp = ag_mfma(at.rows(V, 32 * u, ks), gf[ks], dp);
        }
        if (k0 + 32 * u + 32 > lo) {
            const int left = vis - (k0 + 32 * u + 4 * g);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) < left ? s[e] : AG_NEG;
        }
    };
    auto sweep = [&](int from, int to, auto step) {
        if (from < to) fetch(K0, V0, from);
        AG_LANDED();
        __syncthreads();
        for (int k0 = from; k0 < to; k0 += 2 * BN) {
            if (k0 + BN < to) fetch(K1, V1, k0 + BN);
            if (k0 < hi) step(K0, V0, k0);
            AG_LANDED();
            __syncthreads();
            if (k0 + BN >= to) break;
            if (k0 + 2 * BN < to) fetch(K0, V0, k0 + 2 * BN);
            if (k0 + BN < hi) step(K1, V1, k0 + BN);
            AG_LANDED();
            __syncthreads();
        }
    };
    if (end <= AG_FEW) {
        float sum = 0.f;
        sweep(0, end, [&](const unsigned char* K, const unsigned char* V, int k0) {
            at.keep();
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                f32x16 s, dp;
                products(K, V, k0, u, s, dp);
#pragma unroll
                for (int e = 0; e < 16; ++e) sum = fmaf(__builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -lse)), dp[e], sum);
            }
        });
        sum += __shfl_xor(sum, 32, 64);
        if (vis > 1) dsum = sum;
    }
    if (valid && g == 0 && sp == 0) a.dsum[li] = dsum;

    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = ag_zero();
    auto step = [&](const unsigned char* K, const unsigned char* V, int k0) {
        at.keep();
#pragma unroll
        for (int u = 0; u < BN / 32; ++u) {
            f32x16 s, dp;
            products(K, V, k0, u, s, dp);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -lse)) * (dp[e] - dsum);
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                const s16x8 f = ag_pack(s, h2);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] = ag_mfma(at.cols(K, 32 * u + 16 * h2, dt), f, acc[dt]);
            }
            __builtin_amdgcn_s_setprio(0);
        }
    };
    sweep(kbeg, kend, step);
    if (!valid) return;
    if (a.nsplit == 1) ag_store_row<DC>(a.dq + row * a.D, acc, a.scale, g, a.D);
    else ag_store_part<DC>(a.ws + ((int64_t)sp * a.B * a.Sq * a.Hq + row) * a.D, acc, g, a.D);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: 4 waves x 32 keys, 32 queries a step (64 for DP = 64, whose steps were shorter than a fetch: 8 x 1000
// ragged tokens 78 -> 57 us), over all query heads of the key head's group (so shared heads' gradients are one fixed-order
// sum: no atomics).  S = Q . K^T, dP = dO . V^T (a lane owns one key), dV^T += dO^T . P, dK^T += Q^T . dS.  nsplit > 1: that
// many workgroups share a tile's (head, query) steps, each writes fp32 sums, and ag_add_kernel adds them in order.
// ---------------------------------------------------------------------------
template <int DP, int DC>
__global__ __launch_bounds__(256, 2) void ag_dkv_kernel(AgArgs a) {
    constexpr int KS = DC / 16, DT = DC / 32, BQ = DP == 64 ? 64 : 32, BM = 128;
    __shared__ __attribute__((aligned(16))) unsigned char Q0[BQ * DP * 2], Q1[BQ * DP * 2], G0[BQ * DP * 2], G1[BQ * DP * 2];
    __shared__ __attribute__((aligned(16))) float LD0[128], LD1[128];      // log-sum-exp (0..), D (64..) of a step's queries
    __shared__ __attribute__((aligned(16))) unsigned char Vimg[DP == 128 ? BM * DP * 2 : 16];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv = a.B * a.Hk, units = gridDim.x / a.ntiles;               // units: nsplit x kv
    const int t = blockIdx.x / units, u = blockIdx.x % units;              // low keys are seen by the most queries
    const int b = u % kv / a.Hk, hk = u % kv % a.Hk, sp = u / kv;
    const int klen = ag_klen(a, b);
    const int jw = t * BM + wave * 32, j = jw + (lane & 31), jc = min(j, a.Sk - 1);
    // first query that sees key j: i + 1 + Sk - Sq > j
    const int off = a.Sk - a.Sq;
    const int begin = a.causal ? max(0, t * BM - off) / BQ * BQ : 0;

    // K rows in registers; V rows too for DP = 64, in LDS for DP = 128 (32 registers more would leave one wave a SIMD).
    // Padded keys: rows of no columns, so nothing is read and zeros take part
    const bool seen = j < klen;
    const int width = seen ? a.D : 0;
    s16x8 kf[KS], vf[DP == 128 ? 1 : KS];
    ag_frags<DC>(kf, a.k + b * a.k_bs + jc * a.k_ss + hk * a.k_hs, g, width);
    if constexpr (DP == 128) {
        AgTile<DP, DC, BM, 256> vt;
        vt.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ss, wave, lane);
        vt.load(Vimg, t * BM, klen, a.D, wave);
    } else ag_frags<DC>(vf, a.v + b * a.v_bs + jc * a.v_ss + hk * a.v_hs, g, width);
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        dk[dt] = ag_zero();
        dv[dt] = ag_zero();
    }
    const int steps = t * BM < klen && begin < a.Sq ? (a.Sq - begin + BQ - 1) / BQ : 0;
    const int64_t total = (int64_t)steps * a.group;
    const int n0 = (int)(total * sp / a.nsplit), n1 = (int)(total * (sp + 1) / a.nsplit);
    AgTile<DP, DC, BQ, 256> qt, gt;
    qt.init(a.q + b * a.q_bs, a.q_ss, wave, lane);
    gt.init(a.dO + (int64_t)b * a.Sq * a.Hq * a.D, (int64_t)a.Hq * a.D, wave, lane);
    const char *qs = qt.base, *gs = gt.base;
    // next step to fetch (head of the group, step), to compute
    int fh = steps ? n0 / steps : 0, fq = steps ? n0 % steps : 0, sq = fq;
    auto fetch = [&](unsigned char* Q, unsigned char* G, float* LD) {
        const int h = hk * a.group + fh, q0 = begin + fq * BQ;
        qt.base = qs + h * a.q_hs * 2;
        gt.base = gs + (int64_t)h * a.D * 2;
        qt.load(Q, q0, a.Sq, a.D, wave);
        gt.load(G, q0, a.Sq, a.D, wave);
        if (wave < 2) {                                // no query: log-sum-exp +inf (P = 0) and D 0
            const float* from = (wave ? a.dsum : a.lse) + ((int64_t)b * a.Hq + h) * a.Sq + q0 + lane;
            if (q0 + lane >= a.Sq) from = wave ? reinterpret_cast<const float*>(&ag_zeros) : &ag_inf;
            __builtin_amdgcn_global_load_lds((ag_glb_void*)from, (ag_lds_void*)(LD + wave * 64), 4, 0, 0);
        }
        if (++fq == steps) {
            fq = 0;
            ++fh;
        }
    };
    AgLane<DP> at;
    at.init(lane);
    auto step = [&](const unsigned char* Q, const unsigned char* G, const float* LD) {
        at.keep();
        const int first = begin + sq * BQ;
        if (++sq == steps) sq = 0;
#pragma unroll
        for (int r0 = 0; r0 < BQ; r0 += 32) {
            const int q0 = first + r0;
            if (a.causal && q0 + 31 + off < jw) continue;                  // none of these queries sees this wave's keys
            f32x16 s = ag_zero(), dp = ag_zero();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = ag_mfma(at.rows(Q, r0, ks), kf[ks], s);
                dp = ag_mfma(at.rows(G, r0, ks), DP == 128 ? at.rows(Vimg, wave * 32, ks) : vf[DP == 128 ? 0 : ks], dp);
            }
            __builtin_amdgcn_s_setprio(1);
            if ((a.causal && q0 + off < jw + 31) || jw + 32 > klen) {      // some (query, key) of the tile is not seen
                const int from = !seen ? 0x7fffffff : a.causal ? j - off - q0 - 4 * g : -1;
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = 8 * (x >> 2) + (x & 3) >= from ? s[x] : AG_NEG;
            }
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(LD + r0 + 8 * rq + 4 * g);
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(LD + 64 + r0 + 8 * rq + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = 4 * rq + e;
                    s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], a.scale_log2e, -l4[e]));
                    dp[x] = s[x] * (dp[x] - d4[e]);
                }
            }
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                const s16x8 pf = ag_pack(s, h2), df = ag_pack(dp, h2);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    dv[dt] = ag_mfma(at.cols(G, r0 + 16 * h2, dt), pf, dv[dt]);
                    dk[dt] = ag_mfma(at.cols(Q, r0 + 16 * h2, dt), df, dk[dt]);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
    };
    if (n0 < n1) fetch(Q0, G0, LD0);
    AG_LANDED();
    __syncthreads();
    for (int n = n0; n < n1; n += 2) {
        if (n + 1 < n1) fetch(Q1, G1, LD1);
        step(Q0, G0, LD0);
        AG_LANDED();
        __syncthreads();
        if (n + 1 >= n1) break;
        if (n + 2 < n1) fetch(Q0, G0, LD0);
        step(Q1, G1, LD1);
        AG_LANDED();
        __syncthreads();
    }
    if (j >= a.Sk) return;
    const int64_t o = (((int64_t)b * a.Sk + j) * a.Hk + hk) * a.D;
    if (a.nsplit == 1) {
        ag_store_row<DC>(a.dk + o, dk, a.scale, g, a.D);
        ag_store_row<DC>(a.dv + o, dv, 1.f, g, a.D);
        return;
    }
    const int64_t n = (int64_t)a.B * a.Sk * a.Hk * a.D;
    ag_store_part<DC>(a.ws + sp * 2 * n + o, dk, g, a.D);
    ag_store_part<DC>(a.ws + sp * 2 * n + n + o, dv, g, a.D);
}

// The parts of a tensor of n elements, `stride` floats apart, added in order, scaled and rounded: 4 elements a thread.
// blockIdx.y 0: first tensor (scaled), 1: second, n floats behind it (dK and dV; dQ alone).
__global__ __launch_bounds__(256) void ag_add_kernel(const float* parts, int nsplit, int64_t n, int64_t stride, float scale,
                                                     u16* o0, u16* o1) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    const float* p = parts + blockIdx.y * n + i;
    f32x4 s = *reinterpret_cast<const f32x4*>(p);
    for (int k = 1; k < nsplit; ++k) s += *reinterpret_cast<const f32x4*>(p + k * stride);
    if (blockIdx.y == 0) s *= scale;
    const u32x2 r = {pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
    *reinterpret_cast<u32x2*>((blockIdx.y ? o1 : o0) + i) = r;
}

// ---------------------------------------------------------------------------
static int ag_check(const AgArgs& a, const int64_t* st, int nst) {
    if (a.B <= 0 || a.Sq <= 0 || a.Sk <= 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hq % a.Hk) return -70;
    if (a.D < 8 || a.D > 128 || a.D % 8) return -70;
    for (int i = 0; i < nst; ++i)
        if (st[i] & 7) return -17;
    for (int i = 1; i < nst; i += 3)
        if (st[i] < 0 || st[i] >= (1 << 25)) return -74;
    if ((int64_t)a.Hq * a.D >= (1 << 25)) return -74;
    return 0;
}

static int ag_grid(int64_t n, int* out) {
    if (n > 0x7fffffff) return -72;
    *out = (int)n;
    return 0;
}

// Workgroups that share a tile (by the whole call's size, so a sequence's sums are grouped by how many others there are, not by
// what they hold): enough for `fill` workgroups, no fewer than `least` steps each.  512 are resident (768 to 1024 of heads to
// 64).  2 x 257 queries on 7000 keys, 32 / 8 heads of 128, forward and join: fill 1 151 us, 512 90 + 12, 1024 90 + 20; one token
// on 8192 keys: fill 1 147 us, 512 9 + 6.  512 tokens, 12 heads of 64, dQ and the sum of its parts: fill 1 14.6 us, 512
// 11.7 + 3.6; forward and join 12.2, 9.9 + 4.4.
static int ag_splits(int64_t grid, int64_t steps, int least, int fill) {
    int64_t n = fill / grid, most = steps / least;
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

// PACK where a 128-row tile of one head's queries would be part empty and the group's rows fill fewer tiles: 64 x 1 token on
// 2048 keys, 32 / 8 heads: 98 us (5.5 TB/s of K and V), head by head 361; 2 x 257 queries on 7000 keys 90 + 12, 109 + 9.
static bool ag_pack_rows(int Sq, int group) {
    return group > 1 && Sq <= 512 && ((int64_t)group * Sq + 127) / 128 < (int64_t)group * ((Sq + 127) / 128);
}

static int64_t ag_dsum_floats(int64_t B, int64_t Sq, int64_t Hq) { return (B * Sq * Hq + 3) / 4 * 4; }

static int ag_fwd_splits(int B, int Sq, int Sk, int Hq, int Hk) {
    const bool pack = ag_pack_rows(Sq, Hq / Hk);
    const int64_t rows = pack ? (int64_t)(Hq / Hk) * Sq : Sq;
    return ag_splits((int64_t)B * (pack ? Hk : Hq) * ((rows + 127) / 128), (Sk + 63) / 64, 4, 512);
}

// Causal tiles differ in length, so the longest should be no more than what a slot gets in all: 8192 tokens, 16 / 4 heads of
// 128, dK/dV and the sum of the parts: fill 512 895 + 13 us, 1024 581 + 22, 2048 591 + 49; unshared 1404.
static int ag_dkv_splits(int B, int Sq, int Sk, int Hq, int Hk, int D, int causal) {
    const int bq = D > 64 ? 32 : 64;
    const int64_t steps = (int64_t)((Sq + bq - 1) / bq) * (Hq / Hk);
    return ag_splits((int64_t)B * Hk * ((Sk - 1) / 128 + 1), steps, 256 / bq, causal ? 1024 : 512);
}

#define AG_BY_WIDTH(X)                                              \
    if (D > 96) { X(128, 128) } else if (D > 64) { X(128, 96) }     \
    else if (D > 32) { X(64, 64) } else { X(64, 32) }

extern "C" {

static int ag_dq_splits(int B, int Sq, int Sk, int Hq) {
    return ag_splits((int64_t)B * Hq * ((Sq - 1) / 128 + 1), (Sk + 63) / 64, 4, 512);
}

// What a call is about, packed by its caller (one pointer is cheaper to hand over than twenty arguments): the element strides
// (batch, token, head) of q, k, v; keys of each sequence or null; sizes.
struct AgCall {
    int64_t st[9];
    const int* kv_len;
    int B, Sq, Sk, Hq, Hk, D, causal;
    float scale;
};
static_assert(sizeof(AgCall) == 112, "packed by the caller");

static AgArgs ag_args(const AgCall& c) {
    AgArgs a{};
    a.q_bs = c.st[0]; a.q_ss = c.st[1]; a.q_hs = c.st[2]; a.k_bs = c.st[3]; a.k_ss = c.st[4]; a.k_hs = c.st[5];
    a.v_bs = c.st[6]; a.v_ss = c.st[7]; a.v_hs = c.st[8];
    a.kv_len = c.kv_len; a.B = c.B; a.Sq = c.Sq; a.Sk = c.Sk; a.Hq = c.Hq; a.Hk = c.Hk; a.D = c.D; a.causal = c.causal;
    a.group = c.Hk > 0 ? c.Hq / c.Hk : 0;
    a.scale = c.scale; a.scale_log2e = c.scale * 1.4426950408889634f;
    return a;
}

static bool ag_aligned(void* const* p, int n, int skip) {
    uintptr_t all = 0;
    for (int i = 0; i < n; ++i) all |= i == skip ? 0 : (uintptr_t)p[i];
    return !(all & 15);
}

// fp32 workspace of the forward (0: none) and of the backward (D per query and head, then the parts), in floats
int64_t dtf_attn_general_fwd_ws(const AgCall* c) {
    const int64_t n = ag_fwd_splits(c->B, c->Sq, c->Sk, c->Hq, c->Hk);
    return n > 1 ? n * c->B * c->Sq * c->Hq * (c->D + 2) : 0;
}

int64_t dtf_attn_general_bwd_ws(const AgCall* c) {
    const int64_t n = ag_dkv_splits(c->B, c->Sq, c->Sk, c->Hq, c->Hk, c->D, c->causal), nq = ag_dq_splits(c->B, c->Sq, c->Sk, c->Hq);
    const int64_t kv = n > 1 ? n * 2 * c->B * c->Sk * c->Hk * c->D : 0, q = nq > 1 ? nq * c->B * c->Sq * c->Hq * c->D : 0;
    return ag_dsum_floats(c->B, c->Sq, c->Hq) + (kv > q ? kv : q);     // (dQ's parts are added before dK's are written)
}

// p: q, k, v, o, lse (fp32), ws (dtf_attn_general_fwd_ws floats, or null)
int dtf_attn_general_fwd(void* const* p, const AgCall* c, hipStream_t stream) {
    DTF_CLEAR_ERRORS();
    AgArgs a = ag_args(*c);
    a.q = (const u16*)p[0]; a.k = (const u16*)p[1]; a.v = (const u16*)p[2]; a.out = (u16*)p[3]; a.lse = (float*)p[4]; a.ws = (float*)p[5];
    const int B = c->B, Sq = c->Sq, Sk = c->Sk, Hq = c->Hq, Hk = c->Hk, D = c->D;
    int rc = ag_check(a, c->st, 9), grid = 0;
    if (rc) return rc;
    if (!ag_aligned(p, 6, 4)) return -16;
    const bool pack = ag_pack_rows(Sq, a.group);
    const int64_t rows = pack ? (int64_t)a.group * Sq : Sq;
    a.ntiles = (int)((rows + 127) / 128);
    a.nsplit = ag_fwd_splits(B, Sq, Sk, Hq, Hk);
    if (a.nsplit > 1 && !a.ws) return -73;
    if ((rc = ag_grid((int64_t)B * (pack ? Hk : Hq) * a.ntiles * a.nsplit, &grid))) return rc;
#define AG_FWD(DP, DC)                                                                                     \
    if (pack) hipLaunchKernelGGL((ag_fwd_kernel<DP, DC, true>), dim3(grid), dim3(256), 0, stream, a);      \
    else hipLaunchKernelGGL((ag_fwd_kernel<DP, DC, false>), dim3(grid), dim3(256), 0, stream, a);
    AG_BY_WIDTH(AG_FWD)
#undef AG_FWD
    DTF_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        const int py = a.nsplit <= 2 ? 2 : a.nsplit <= 4 ? 4 : 8;
        if ((rc = ag_grid(((int64_t)B * Sq * Hq * py + 7) / 8, &grid))) return rc;
        if (py == 2) hipLaunchKernelGGL((ag_join_kernel<2>), dim3(grid), dim3(256), 0, stream, a);
        else if (py == 4) hipLaunchKernelGGL((ag_join_kernel<4>), dim3(grid), dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((ag_join_kernel<8>), dim3(grid), dim3(256), 0, stream, a);
        DTF_CHECK_LAUNCH();
    }
    return 0;
}

// p: q, k, v, o, dO, lse, dq, dk, dv, ws (dtf_attn_general_bwd_ws floats); o, dO, dq contiguous [B, Sq, Hq, D], dk, dv
// contiguous [B, Sk, Hk, D]
int dtf_attn_general_bwd(void* const* p, const AgCall* c, hipStream_t stream) {
    DTF_CLEAR_ERRORS();
    AgArgs a = ag_args(*c);
    const int B = c->B, Sq = c->Sq, Sk = c->Sk, Hq = c->Hq, Hk = c->Hk, D = c->D, causal = c->causal;
    const float scale = c->scale;
    float* ws = (float*)p[9];
    a.q = (const u16*)p[0]; a.k = (const u16*)p[1]; a.v = (const u16*)p[2]; a.o = (const u16*)p[3]; a.dO = (const u16*)p[4];
    a.lse = (float*)p[5]; a.dq = (u16*)p[6]; a.dk = (u16*)p[7]; a.dv = (u16*)p[8]; a.dsum = ws;
    int rc = ag_check(a, c->st, 9), grid = 0;
    if (rc) return rc;
    if (!ag_aligned(p, 10, 5)) return -16;
    a.ws = ws + ag_dsum_floats(B, Sq, Hq);
    const int splits = ag_dkv_splits(B, Sq, Sk, Hq, Hk, D, causal);
    if (!ws) return -73;
    if ((int64_t)((Sq + 31) / 32) * a.group > 0x7fffffff) return -72;
    a.ntiles = (Sq - 1) / 128 + 1;
    a.nsplit = ag_dq_splits(B, Sq, Sk, Hq);
    if ((rc = ag_grid((int64_t)B * Hq * a.ntiles * a.nsplit, &grid))) return rc;
#define AG_DQ(DP, DC) hipLaunchKernelGGL((ag_dq_kernel<DP, DC>), dim3(grid), dim3(256), 0, stream, a);
    AG_BY_WIDTH(AG_DQ)
#undef AG_DQ
    DTF_CHECK_LAUNCH();
    if (a.nsplit > 1) {
        const int64_t n = (int64_t)B * Sq * Hq * D;
        if ((rc = ag_grid((n + 1023) / 1024, &grid))) return rc;
        hipLaunchKernelGGL(ag_add_kernel, dim3(grid), dim3(256), 0, stream, a.ws, a.nsplit, n, n, scale, a.dq, (u16*)nullptr);
        DTF_CHECK_LAUNCH();
    }
    a.ntiles = (Sk - 1) / 128 + 1;
    a.nsplit = splits;
    if ((rc = ag_grid((int64_t)B * Hk * a.ntiles * splits, &grid))) return rc;
#define AG_DKV(DP, DC) hipLaunchKernelGGL((ag_dkv_kernel<DP, DC>), dim3(grid), dim3(256), 0, stream, a);
    AG_BY_WIDTH(AG_DKV)
#undef AG_DKV
    DTF_CHECK_LAUNCH();
    if (splits > 1) {
        const int64_t n = (int64_t)B * Sk * Hk * D;
        if ((rc = ag_grid((n + 1023) / 1024, &grid))) return rc;
        hipLaunchKernelGGL(ag_add_kernel, dim3(grid, 2), dim3(256), 0, stream, a.ws, splits, n, 2 * n, scale, a.dk, a.dv);
        DTF_CHECK_LAUNCH();
    }
    return 0;
}

}  // extern "C"
