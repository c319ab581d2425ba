// Self-attention with score modifiers for gfx950: grouped key heads, a tanh cap, a bias that falls with the distance,
// document masks and visible prefixes, forward and backward, bf16 with fp32 statistics and accumulators.
//
//   x_ij = scale q_i . k_j,   x <- cap tanh(x / cap),   x <- x - slope_h |i - j|,
//   visible(i, j) = (j <= i or j < prefix or not causal) and doc_i == doc_j >= 0,
//   P = softmax over the visible j,   O = P V;   a row that sees nothing has O = 0 and no gradient.
//   dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta) (1 - tanh^2) scale,  dQ = dS K, dK = dS^T Q, dV = P^T dO.
//
// Same arrangement as attention.hip (transposed score tile S^T = K Q^T, so that a query's statistics sit on one lane and
// the score registers are the B operand of the next product; see attn_tile.h).  What is new:
//   * Which 64-row tiles a workgroup visits is decided from the smallest and largest document number of every 32 rows
//     (one small kernel ahead): 64 tiles are tested at a time, one per lane, and the ballot is walked bit by bit.  Any
//     numbering is right - ranges that overlap are visited and masked element by element -, sorted ones are fast.
//   * Scores are kept in the exponent's base 2 throughout; tanh(x) = 1 - 2 r with r = 1 / (1 + e^{2x}), so that
//     1 - tanh^2 = 4 r (1 - r) costs no second transcendental in the backward kernels.
//   * delta comes from the same MFMA as dP (the diagonal of O dO^T): a row with one visible key has dP = delta bit for
//     bit, and its dS is exactly zero as the formula says.  O enters it with what its rounding took away (kept by the
//     forward in bf16, `rest`): where a few keys carry a row, dS is a small difference of dP and delta, and delta from the
//     rounded O alone costs dQ and dK as much accuracy as their own rounding does (3.8e-3 against 2.5e-3 of the norm at
//     scores of standard deviation 8 under a cap of 30).
//   * Rows behind a document number < 0 are staged as zeros: whatever a padded row holds reaches no product.
#include <math.h>
#include "attn_tile.h"
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

using namespace attn;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float MASKED = -2.0e30f;       // below every running maximum (which starts at NEG_BIG): exp2 gives 0 even in a row without keys
constexpr int BQ = 128;                  // rows of a workgroup

struct DocRange { int lo, hi; };         // of 32 or more rows; padded rows count as -1

__device__ __forceinline__ DocRange merge(DocRange a, DocRange b) { return {min(a.lo, b.lo), max(a.hi, b.hi)}; }
__device__ __forceinline__ bool meets(DocRange a, DocRange b) { return a.hi >= 0 && b.hi >= 0 && max(a.lo, 0) <= b.hi && max(b.lo, 0) <= a.hi; }
__device__ __forceinline__ bool same_doc(DocRange a, DocRange b) { return a.lo >= 0 && a.lo == a.hi && b.lo == b.hi && a.lo == b.lo; }

// ranges[b][t] = (lo, hi) of rows 64 t .. 64 t + 31 and of the 32 behind them
__global__ __launch_bounds__(256) void doc_ranges_kernel(const int* __restrict__ docs, int4* __restrict__ ranges, int T, int tiles) {
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= tiles) return;
    const int row = t * 64 + lane;
    int lo = 0x7fffffff, hi = -0x7fffffff;
    if (row < T) lo = hi = max(docs[(long)blockIdx.y * T + row], -1);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        lo = min(lo, __shfl_xor(lo, off, 64));
        hi = max(hi, __shfl_xor(hi, off, 64));
    }
    const int lo2 = __shfl(lo, 32, 64), hi2 = __shfl(hi, 32, 64);
    if (lane == 0) ranges[(long)blockIdx.y * tiles + t] = make_int4(lo, hi, lo2, hi2);
}

// document range of rows r0 .. r0 + 32 n - 1 (r0 a multiple of 32, ends past the last tile left out)
__device__ __forceinline__ DocRange range_of(const int4* rg, int r0, int n, int tiles) {
    DocRange d{0x7fffffff, -0x7fffffff};
    for (int i = 0; i < n; ++i) {
        const int g = (r0 >> 5) + i;
        if ((g >> 1) >= tiles) break;
        const int4 v = rg[g >> 1];
        d = merge(d, (g & 1) ? DocRange{v.z, v.w} : DocRange{v.x, v.y});
    }
    return d;
}

// Walks the 64-row tiles first .. end - 1 that a workgroup's rows can share a document with.  `mine` / `whole`: whether the
// wave's own 32 rows meet the current tile, and whether every pair of the two is of one document.
struct TileWalk {
    const int4* rg;                      // nullptr: no documents, every tile is visited whole
    int base, end, j;
    DocRange block, wave;
    unsigned long long todo, mine_bits, whole_bits;
    bool mine, whole;

    __device__ __forceinline__ void look() {
        const int lane = threadIdx.x & 63, t = base + lane;
        bool a = t < end, b = true, c = true;
        if (rg != nullptr) {
            DocRange d{0x7fffffff, -0x7fffffff};
            if (a) {
                const int4 v = rg[t];
                d = merge(DocRange{v.x, v.y}, DocRange{v.z, v.w});
            }
            a = a && meets(d, block);
            b = meets(d, wave);
            c = same_doc(d, wave);
        }
        todo = __ballot(a); mine_bits = __ballot(b); whole_bits = __ballot(c);
    }
    __device__ __forceinline__ void start(int first, int end_) { base = first; end = end_; look(); }
    // the next tile, or `end` when there is none
    __device__ __forceinline__ int next() {
        while (todo == 0) {
            base += 64;
            if (base >= end) { base = end; return end; }
            look();
        }
        const int bit = __ffsll((long long)todo) - 1;
        todo &= todo - 1;
        mine = (mine_bits >> bit) & 1; whole = (whole_bits >> bit) & 1;
        return base + bit;
    }
};

// A 64 x DH tile on its way to LDS.  Rows past T and rows of padding become zeros; columns past D repeat the last eight (the
// other operand of every product that sums over them is zero there).
template <int DH>
struct Staged {
    u32x4 r[DH / 32];
    int doc[DH / 32];
    __device__ __forceinline__ void fetch(const unsigned short* __restrict__ g, long rs, int r0, int T, int D, const int* __restrict__ docs, int tid) {
        constexpr int CPR = DH / 8, RSTEP = 256 / CPR;
        const int col = min((tid % CPR) * 8, D - 8);
#pragma unroll
        for (int i = 0; i < DH / 32; ++i) {
            const int row = r0 + tid / CPR + i * RSTEP, rc = min(row, T - 1);
            r[i] = *(const u32x4*)(g + (long)rc * rs + col);
            doc[i] = row < T ? (docs != nullptr ? docs[rc] : 0) : -1;
        }
    }
    __device__ __forceinline__ void stash(unsigned char* lds, int tid) const {
        constexpr int CPR = DH / 8, RSTEP = 256 / CPR;
        const int c = tid % CPR;
#pragma unroll
        for (int i = 0; i < DH / 32; ++i)
            *(u32x4*)(lds + img_off<DH>(tid / CPR + i * RSTEP, c * 8)) = doc[i] < 0 ? u32x4{0, 0, 0, 0} : r[i];
    }
};

// this lane's half of one row as MFMA fragments, zero from column D on (and everywhere unless `live`)
template <int DH>
__device__ __forceinline__ void load_frags(const unsigned short* row, int h, int D, bool live, bf16x8 (&f)[DH / 16]) {
#pragma unroll
    for (int kk = 0; kk < DH / 16; ++kk) {
        const int col = 16 * kk + 8 * h;
        u32x4 v = {0, 0, 0, 0};
        if (live && col < D) v = *(const u32x4*)(row + col);
        f[kk] = __builtin_bit_cast(bf16x8, v);
    }
}

template <int DH>
__device__ __forceinline__ void store_cols(unsigned short* __restrict__ dst, const floatx16 (&acc)[DH / 32], float scale, int h, int D) {
#pragma unroll
    for (int di = 0; di < DH / 32; ++di)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * di + 8 * g + 4 * h;
            if (d < D) {
                uint2 pk;
                pk.x = pack_bf16x2(acc[di][4 * g + 0] * scale, acc[di][4 * g + 1] * scale);
                pk.y = pack_bf16x2(acc[di][4 * g + 2] * scale, acc[di][4 * g + 3] * scale);
                *(uint2*)(dst + d) = pk;
            }
        }
}

// score of a pair in base 2 from the raw product; `r` (cap only): 1 / (1 + e^{2x}), from which 1 - tanh^2 = 4 r (1 - r)
struct ScoreMap { float c, k1, cap2; };       // scale log2 e;  2 scale log2 e / cap;  cap log2 e
template <bool CAP>
__device__ __forceinline__ float map_score(const ScoreMap& m, float s, float& r) {
    if (CAP) {
        r = __builtin_amdgcn_rcpf(1.f + fast_exp2(s * m.k1));
        return fmaf(r, -2.f * m.cap2, m.cap2);
    }
    return s * m.c;
}

// ------------------------------------------------------------------------------ forward
template <int DH, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, DH == 64 ? 2 : 1) void attend_fwd_kernel(AttendArgs a, unsigned short* __restrict__ out, unsigned short* __restrict__ rest, float* __restrict__ lse2) {
    constexpr int KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>();
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * TB + TILE * 4];
    unsigned char* Ks = smem;
    unsigned char* Vs = smem + TB;
    int* Kd = (int*)(smem + 2 * TB);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ql = lane & 31, h = lane >> 5;
    const int head = blockIdx.x, b = blockIdx.y, hk = head / (a.Hq / a.Hkv);
    const int T = a.T, q0 = (gridDim.z - 1 - blockIdx.z) * BQ, qw0 = q0 + 32 * wave, q = qw0 + ql, qc = min(q, T - 1);
    const unsigned short* qbase = (const unsigned short*)a.q + b * a.qb + head * a.qh;
    const unsigned short* kbase = (const unsigned short*)a.k + b * a.kb + hk * a.kh;
    const unsigned short* vbase = (const unsigned short*)a.v + b * a.vb + hk * a.vh;
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = a.causal ? (a.prefix != nullptr ? min(max(a.prefix[b], 0), T) : 0) : T;
    const int lim = max(qc, pre - 1);                               // the last key that this lane's query sees
    const int qdoc = docs != nullptr ? docs[qc] : 0;
    const ScoreMap sm{a.scale * LOG2E, CAP ? 2.f * a.scale / a.softcap * LOG2E : 0.f, a.softcap * LOG2E};
    const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;

    bf16x8 qf[KK];
    load_frags<DH>(qbase + (long)qc * a.qt, h, a.D, qdoc >= 0, qf);

    TileWalk walk;
    walk.rg = docs != nullptr ? a.ranges + (long)b * tiles : nullptr;
    if (docs != nullptr) {
        walk.block = range_of(walk.rg, q0, BQ / 32, tiles);
        walk.wave = range_of(walk.rg, qw0, 1, tiles);
    }
    walk.start(0, max(min(q0 + BQ, T), pre) / TILE + (max(min(q0 + BQ, T), pre) % TILE != 0));
    const int wave_last = max(min(qw0 + 31, T - 1), pre - 1), wave_least = max(min(qw0, T - 1), pre - 1);

    floatx16 O[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) zero16(O[di]);
    float m = NEG_BIG, l = 0.f;
    Staged<DH> pk, pv;
    int kd = 0;
    int j = walk.next();
    bool mine = walk.mine, whole = walk.whole;
    if (j < walk.end) {
        pk.fetch(kbase, a.kt, j * TILE, T, a.D, docs, tid);
        pv.fetch(vbase, a.vt, j * TILE, T, a.D, docs, tid);
        if (docs != nullptr && tid < TILE) kd = docs[min(j * TILE + tid, T - 1)];
    }
    while (j < walk.end) {
        __syncthreads();
        pk.stash(Ks, tid);
        pv.stash(Vs, tid);
        if (docs != nullptr && tid < TILE) Kd[tid] = kd;
        __syncthreads();
        const int jt = j * TILE;
        const bool go = mine && jt <= wave_last, same = whole, full = same && jt + TILE - 1 <= wave_least;
        j = walk.next();
        mine = walk.mine; whole = walk.whole;
        if (j < walk.end) {
            pk.fetch(kbase, a.kt, j * TILE, T, a.D, docs, tid);
            pv.fetch(vbase, a.vt, j * TILE, T, a.D, docs, tid);
            if (docs != nullptr && tid < TILE) kd = docs[min(j * TILE + tid, T - 1)];
        }
        if (!go) continue;                                          // wave-uniform
        floatx16 S[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            zero16(S[t2]);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                S[t2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<DH>(Ks, 32 * t2 + ql, kk, h), qf[kk], S[t2], 0, 0, 0);
        }
        float mx = NEG_BIG;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float rr;
                float y = (CAP || BIAS) ? map_score<CAP>(sm, S[t2][r], rr) : S[t2][r];
                if (BIAS) y = fmaf(-slope2, fabsf((float)(q - jt - 4 * h) - (float)(32 * t2 + acc_row(r, 0))), y);
                if (!full) {                                        // wave-uniform
                    const int key = 32 * t2 + acc_row(r, h);
                    const bool see = jt + key <= lim && (same || Kd[key] == qdoc);
                    y = see ? y : MASKED;
                }
                S[t2][r] = y;
                mx = fmaxf(mx, y);
            }
        mx = xhalf_max(mx);
        const float c = (CAP || BIAS) ? 1.f : sm.c;                 // the scale rides the exponent's multiply-add where nothing else used it
        const float mn = fmaxf(m, mx * c);
        const bool grew = mn > m;
        float rsum = 0.f;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = fast_exp2((CAP || BIAS) ? S[t2][r] - mn : fmaf(S[t2][r], c, -mn));
                S[t2][r] = p;
                rsum += p;
            }
        rsum = xhalf_sum(rsum);
        if (__any(grew)) {
            const float alpha = fast_exp2(m - mn);
            l *= alpha;
#pragma unroll
            for (int di = 0; di < DI; ++di)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[di][r] *= alpha;
        }
        l += rsum;
        m = mn;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 pb = pack_regs(S[t2], s);
#pragma unroll
                for (int di = 0; di < DI; ++di)
                    O[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag<DH>(Vs, 32 * t2 + 16 * s + 4 * h, 32 * di, lane), pb,
                                                                    O[di], 0, 0, 0);
            }
    }
    if (q < T) {
        const bool empty = l == 0.f;                                // saw no key: output zero, and P = exp2(x - 1e30) = 0 in backward
        // a sum this near 1 is one key's exponent off by its own rounding: taken as 1, so that O is that key's V exactly
        const bool one = fabsf(l - 1.f) <= 2.384185791015625e-7f * fmaxf(1.f, fabsf(m));
        const float inv = empty ? 0.f : one ? 1.f : 1.f / l;
        const long row = (((long)b * T + q) * a.Hq + head) * a.D;
#pragma unroll
        for (int di = 0; di < DI; ++di)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[di][r] *= inv;
        store_cols<DH>(out + row, O, 1.f, h, a.D);
        if (rest != nullptr) {
#pragma unroll
            for (int di = 0; di < DI; ++di)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[di][r] -= bf16_to_float(float_to_bf16(O[di][r]));
            store_cols<DH>(rest + row, O, 1.f, h, a.D);
        }
        if (h == 0) lse2[((long)b * a.Hq + head) * T + q] = empty ? 1.0e30f : m + __log2f(l);
    }
}

// ------------------------------------------------------------------------------ dQ (query-stationary), and delta
template <int DH, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, DH == 64 ? 2 : 1) void attend_bwd_q_kernel(AttendArgs a, const unsigned short* __restrict__ out, const unsigned short* __restrict__ rest,
                                                                            const unsigned short* __restrict__ dout, const float* __restrict__ lse2,
                                                                            float* __restrict__ delta, unsigned short* __restrict__ dq) {
    constexpr int KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>();
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * TB + TILE * 4];
    unsigned char* Ks = smem;
    unsigned char* Vs = smem + TB;
    int* Kd = (int*)(smem + 2 * TB);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ql = lane & 31, h = lane >> 5;
    const int head = blockIdx.x, b = blockIdx.y, hk = head / (a.Hq / a.Hkv);
    const int T = a.T, q0 = (gridDim.z - 1 - blockIdx.z) * BQ, qw0 = q0 + 32 * wave, q = qw0 + ql, qc = min(q, T - 1);
    const unsigned short* qbase = (const unsigned short*)a.q + b * a.qb + head * a.qh;
    const unsigned short* kbase = (const unsigned short*)a.k + b * a.kb + hk * a.kh;
    const unsigned short* vbase = (const unsigned short*)a.v + b * a.vb + hk * a.vh;
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = a.causal ? (a.prefix != nullptr ? min(max(a.prefix[b], 0), T) : 0) : T;
    const int lim = max(qc, pre - 1);
    const int qdoc = docs != nullptr ? docs[qc] : 0;
    const ScoreMap sm{a.scale * LOG2E, CAP ? 2.f * a.scale / a.softcap * LOG2E : 0.f, a.softcap * LOG2E};
    const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
    const long orow = (((long)b * T + qc) * a.Hq + head) * a.D;

    bf16x8 qf[KK], dof[KK];
    load_frags<DH>(qbase + (long)qc * a.qt, h, a.D, qdoc >= 0, qf);
    load_frags<DH>(dout + orow, h, a.D, qdoc >= 0, dof);
    float del;
    {
        bf16x8 of[KK];
        load_frags<DH>(out + orow, h, a.D, qdoc >= 0, of);
        floatx16 dd;
        zero16(dd);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) dd = __builtin_amdgcn_mfma_f32_32x32x16_bf16(of[kk], dof[kk], dd, 0, 0, 0);
        load_frags<DH>(rest + orow, h, a.D, qdoc >= 0, of);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) dd = __builtin_amdgcn_mfma_f32_32x32x16_bf16(of[kk], dof[kk], dd, 0, 0, 0);
        del = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) del = acc_row(r, h) == ql ? dd[r] : del;
        del = xhalf_sum(del);                                       // one half holds the diagonal element, the other zero
    }
    if (h == 0 && q < T) delta[((long)b * a.Hq + head) * T + q] = del;
    const float lse_q = lse2[((long)b * a.Hq + head) * T + qc];

    TileWalk walk;
    walk.rg = docs != nullptr ? a.ranges + (long)b * tiles : nullptr;
    if (docs != nullptr) {
        walk.block = range_of(walk.rg, q0, BQ / 32, tiles);
        walk.wave = range_of(walk.rg, qw0, 1, tiles);
    }
    walk.start(0, max(min(q0 + BQ, T), pre) / TILE + (max(min(q0 + BQ, T), pre) % TILE != 0));
    const int wave_last = max(min(qw0 + 31, T - 1), pre - 1), wave_least = max(min(qw0, T - 1), pre - 1);

    floatx16 dQt[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) zero16(dQt[di]);
    Staged<DH> pk, pv;
    int kd = 0;
    int j = walk.next();
    bool mine = walk.mine, whole = walk.whole;
    if (j < walk.end) {
        pk.fetch(kbase, a.kt, j * TILE, T, a.D, docs, tid);
        pv.fetch(vbase, a.vt, j * TILE, T, a.D, docs, tid);
        if (docs != nullptr && tid < TILE) kd = docs[min(j * TILE + tid, T - 1)];
    }
    while (j < walk.end) {
        __syncthreads();
        pk.stash(Ks, tid);
        pv.stash(Vs, tid);
        if (docs != nullptr && tid < TILE) Kd[tid] = kd;
        __syncthreads();
        const int jt = j * TILE;
        const bool go = mine && jt <= wave_last, same = whole;
        j = walk.next();
        mine = walk.mine; whole = walk.whole;
        if (j < walk.end) {
            pk.fetch(kbase, a.kt, j * TILE, T, a.D, docs, tid);
            pv.fetch(vbase, a.vt, j * TILE, T, a.D, docs, tid);
            if (docs != nullptr && tid < TILE) kd = docs[min(j * TILE + tid, T - 1)];
        }
        if (!go) continue;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const int kt0 = jt + 32 * t2;
            if (kt0 > wave_last) continue;                          // wave-uniform
            const bool full = same && kt0 + 31 <= wave_least;
            floatx16 S, dP;
            zero16(S); zero16(dP);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<DH>(Ks, 32 * t2 + ql, kk, h), qf[kk], S, 0, 0, 0);
                dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<DH>(Vs, 32 * t2 + ql, kk, h), dof[kk], dP, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float rr = 0.f;
                float y = map_score<CAP>(sm, S[r], rr);
                if (BIAS) y = fmaf(-slope2, fabsf((float)(q - kt0 - 4 * h) - (float)acc_row(r, 0)), y);
                const float p = fast_exp2(y - lse_q);
                float ds = p * a.scale * (dP[r] - del);
                if (CAP) ds *= 4.f * rr * (1.f - rr);
                if (!full) {
                    const int key = acc_row(r, h);
                    const bool see = kt0 + key <= lim && (same || Kd[32 * t2 + key] == qdoc);
                    ds = see ? ds : 0.f;
                }
                S[r] = ds;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 dsb = pack_regs(S, s);
#pragma unroll
                for (int di = 0; di < DI; ++di)
                    dQt[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag<DH>(Ks, 32 * t2 + 16 * s + 4 * h, 32 * di, lane), dsb,
                                                                      dQt[di], 0, 0, 0);
            }
        }
    }
    if (q < T) store_cols<DH>(dq + orow, dQt, qdoc >= 0 ? 1.f : 0.f, h, a.D);
}

// ------------------------------------------------------------------------------ dK / dV (key-stationary, no atomics)
template <int DH, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, DH == 64 ? 2 : 1) void attend_bwd_kv_kernel(AttendArgs a, const unsigned short* __restrict__ dout,
                                                                             const float* __restrict__ lse2, const float* __restrict__ delta,
                                                                             unsigned short* __restrict__ dk, unsigned short* __restrict__ dv) {
    constexpr int KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>();
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * TB + 3 * TILE * 4];
    unsigned char* Qs = smem;
    unsigned char* Os = smem + TB;
    float* lse_s = (float*)(smem + 2 * TB);
    float* del_s = lse_s + TILE;
    int* Qd = (int*)(del_s + TILE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kl = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x, b = blockIdx.y, group = a.Hq / a.Hkv;
    const int T = a.T, k0 = blockIdx.z * BQ, kw0 = k0 + 32 * wave, key = kw0 + kl, keyc = min(key, T - 1);
    const unsigned short* kbase = (const unsigned short*)a.k + b * a.kb + hk * a.kh;
    const unsigned short* vbase = (const unsigned short*)a.v + b * a.vb + hk * a.vh;
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = a.causal ? (a.prefix != nullptr ? min(max(a.prefix[b], 0), T) : 0) : T;
    const int kdoc = docs != nullptr ? docs[keyc] : 0;
    const ScoreMap sm{a.scale * LOG2E, CAP ? 2.f * a.scale / a.softcap * LOG2E : 0.f, a.softcap * LOG2E};

    bf16x8 kf[KK], vf[KK];
    load_frags<DH>(kbase + (long)keyc * a.kt, h, a.D, kdoc >= 0, kf);
    load_frags<DH>(vbase + (long)keyc * a.vt, h, a.D, kdoc >= 0, vf);
    floatx16 dKt[DI], dVt[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) { zero16(dKt[di]); zero16(dVt[di]); }

    TileWalk walk;
    walk.rg = docs != nullptr ? a.ranges + (long)b * tiles : nullptr;
    if (docs != nullptr) {
        walk.block = range_of(walk.rg, k0, BQ / 32, tiles);
        walk.wave = range_of(walk.rg, kw0, 1, tiles);
    }
    const int first = k0 < pre ? 0 : k0 / TILE;                     // in front of the first key only a prefix key is seen
    const int key_from = key < pre ? -(1 << 30) : key;              // the first query that sees this lane's key

    for (int g = 0; g < group; ++g) {
        const int head = hk * group + g;
        const unsigned short* qbase = (const unsigned short*)a.q + b * a.qb + head * a.qh;
        const unsigned short* dobase = dout + ((long)b * T * a.Hq + head) * a.D;
        const float* lse_b = lse2 + ((long)b * a.Hq + head) * T;
        const float* del_b = delta + ((long)b * a.Hq + head) * T;
        const long ors = (long)a.Hq * a.D;
        const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
        Staged<DH> pq, po;
        float pl = 0.f, pd = 0.f;
        int pdoc = 0;
        walk.start(first, tiles);
        int j = walk.next();
        bool mine = walk.mine, whole = walk.whole;
#define DPA_FETCH_Q()                                                                  \
    if (j < walk.end) {                                                                \
        pq.fetch(qbase, a.qt, j * TILE, T, a.D, docs, tid);                            \
        po.fetch(dobase, ors, j * TILE, T, a.D, docs, tid);                            \
        if (tid < TILE) {                                                              \
            const int qi = j * TILE + tid;                                             \
            pl = qi < T ? lse_b[qi] : 1.0e30f;                                         \
            pd = qi < T ? del_b[qi] : 0.f;                                             \
            pdoc = docs != nullptr && qi < T ? docs[qi] : 0;                           \
        }                                                                              \
    }
        DPA_FETCH_Q()
        while (j < walk.end) {
            __syncthreads();
            pq.stash(Qs, tid);
            po.stash(Os, tid);
            if (tid < TILE) { lse_s[tid] = pl; del_s[tid] = pd; Qd[tid] = pdoc; }
            __syncthreads();
            const int jt = j * TILE;
            const bool go = mine && (jt + TILE - 1 >= kw0 || kw0 < pre), same = whole;
            j = walk.next();
            mine = walk.mine; whole = walk.whole;
            DPA_FETCH_Q()
            if (!go) continue;                                      // wave-uniform
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const int qt0 = jt + 32 * t2;
                if (qt0 + 31 < kw0 && kw0 >= pre) continue;         // wave-uniform
                const bool full = same && (qt0 >= kw0 + 31 || kw0 + 31 < pre);
                floatx16 S, dP;
                zero16(S); zero16(dP);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<DH>(Qs, 32 * t2 + kl, kk, h), kf[kk], S, 0, 0, 0);
                    dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<DH>(Os, 32 * t2 + kl, kk, h), vf[kk], dP, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int qr = 32 * t2 + acc_row(r, h);
                    float rr = 0.f;
                    float y = map_score<CAP>(sm, S[r], rr);
                    if (BIAS) y = fmaf(-slope2, fabsf((float)(qt0 + 4 * h - key) + (float)acc_row(r, 0)), y);
                    float p = fast_exp2(y - lse_s[qr]);
                    float ds = p * a.scale * (dP[r] - del_s[qr]);
                    if (CAP) ds *= 4.f * rr * (1.f - rr);
                    if (!full) {
                        const bool see = jt + qr >= key_from && (same || Qd[qr] == kdoc);
                        p = see ? p : 0.f;
                        ds = see ? ds : 0.f;
                    }
                    S[r] = p;
                    dP[r] = ds;
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 pb = pack_regs(S, s), dsb = pack_regs(dP, s);
                    const int rowbase = 32 * t2 + 16 * s + 4 * h;
#pragma unroll
                    for (int di = 0; di < DI; ++di) {
                        dVt[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag<DH>(Os, rowbase, 32 * di, lane), pb, dVt[di], 0, 0, 0);
                        dKt[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag<DH>(Qs, rowbase, 32 * di, lane), dsb, dKt[di], 0, 0, 0);
                    }
                }
            }
        }
#undef DPA_FETCH_Q
    }
    if (key < T) {
        const long row = (((long)b * T + key) * a.Hkv + hk) * a.D;
        store_cols<DH>(dk + row, dKt, kdoc >= 0 ? 1.f : 0.f, h, a.D);
        store_cols<DH>(dv + row, dVt, kdoc >= 0 ? 1.f : 0.f, h, a.D);
    }
}

template <int DH, bool CAP, bool BIAS>
void fwd_of(const AttendArgs& a, void* out, void* rest, float* lse2, hipStream_t st) {
    hipLaunchKernelGGL((attend_fwd_kernel<DH, CAP, BIAS>), dim3(a.Hq, a.B, (a.T + BQ - 1) / BQ), dim3(256), 0, st, a, (unsigned short*)out,
                       (unsigned short*)rest, lse2);
}
template <int DH, bool CAP, bool BIAS>
void bwd_of(const AttendArgs& a, const void* out, const void* rest, const void* dout, const float* lse2, float* delta, void* dq, void* dk, void* dv, hipStream_t st) {
    const int blocks = (a.T + BQ - 1) / BQ;
    hipLaunchKernelGGL((attend_bwd_q_kernel<DH, CAP, BIAS>), dim3(a.Hq, a.B, blocks), dim3(256), 0, st, a, (const unsigned short*)out,
                       (const unsigned short*)rest, (const unsigned short*)dout, lse2, delta, (unsigned short*)dq);
    hipLaunchKernelGGL((attend_bwd_kv_kernel<DH, CAP, BIAS>), dim3(a.Hkv, a.B, blocks), dim3(256), 0, st, a, (const unsigned short*)dout,
                       lse2, delta, (unsigned short*)dk, (unsigned short*)dv);
}

}  // namespace

// one build per (width, cap, bias): the masks are wave-uniform branches inside
#define DPA_ATTEND_PICK(F, ...)                                                                                         \
    do {                                                                                                                \
        const bool cap = a.softcap > 0.f, bias = a.slopes != nullptr;                                                   \
        if (a.D <= 64) {                                                                                                \
            if (cap) { if (bias) F<64, true, true>(__VA_ARGS__); else F<64, true, false>(__VA_ARGS__); }                \
            else { if (bias) F<64, false, true>(__VA_ARGS__); else F<64, false, false>(__VA_ARGS__); }                  \
        } else {                                                                                                        \
            if (cap) { if (bias) F<128, true, true>(__VA_ARGS__); else F<128, true, false>(__VA_ARGS__); }              \
            else { if (bias) F<128, false, true>(__VA_ARGS__); else F<128, false, false>(__VA_ARGS__); }                \
        }                                                                                                               \
    } while (0)

void attend_doc_ranges(const int* docs, void* ranges, int B, int T, hipStream_t st) {
    const int tiles = (T + TILE - 1) / TILE;
    hipLaunchKernelGGL(doc_ranges_kernel, dim3((tiles + 3) / 4, B), dim3(256), 0, st, docs, (int4*)ranges, T, tiles);
}

void attend_fwd(const AttendArgs& a, void* out, void* rest, float* lse2, hipStream_t st) { DPA_ATTEND_PICK(fwd_of, a, out, rest, lse2, st); }

void attend_bwd(const AttendArgs& a, const void* out, const void* rest, const void* dout, const float* lse2, float* delta, void* dq, void* dk, void* dv, hipStream_t st) {
    DPA_ATTEND_PICK(bwd_of, a, out, rest, dout, lse2, delta, dq, dk, dv, st);
}

}  // namespace dpa
