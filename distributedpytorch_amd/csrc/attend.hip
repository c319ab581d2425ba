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
//     1 - tanh^2 = 4 r (e^{2x} r) costs no second transcendental in the backward kernels.  Near x = 0 that difference cancels
//     and leaves the score some 1.8e-7 of the cap off: caps past CAP_MOST take a build with a relative error instead.
//   * delta comes from the same MFMA as dP (the diagonal of O dO^T): a row with one visible key has dP = delta bit for
//     bit, and its dS is exactly zero as the formula says.  O enters it with what its rounding took away (kept by the
//     forward in bf16, `rest`): where a few keys carry a row, dS is a small difference of dP and delta, and delta from the
//     rounded O alone costs dQ and dK as much accuracy as their own rounding does (3.8e-3 against 2.5e-3 of the norm at
//     scores of standard deviation 8 under a cap of 30).
//   * Rows behind a document number < 0 are staged as zeros, so that whatever a padded row holds reaches no sum (the values that the
//     dK / dV kernel of width 128 keeps are not: a padded key's reach its own column of dP alone, which its mask zeroes).
//
// Bound by the matrix cores and the vector instructions between their products (exponentials, masks, rounding), which a wave
// does not overlap by itself.  One row of 8192, 16 query heads over 4 of width 128, with a bias: forward 347 us (790 TFLOP/s of
// the visible half), dQ 367 (1120), dK / dV 500 + 23 for the parts (1050); a large matrix product reaches 1230 here.  Short
// documents are bound by the tiles at their edges instead: 16 rows of 1024 in documents of 256, 12 heads of width 64: 52 / 51 /
// 56 us, where their traffic alone would take 26 / 37 / 31.
#include <math.h>
#include <type_traits>
#include "attn_tile.h"
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

using namespace attn;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float MASKED = -2.0e30f;       // below every running maximum (which starts at NEG_BIG): exp2 gives 0 even in a row without keys
constexpr int BQ = 128;                  // rows of a workgroup
// The kernels' builds by cap: none, one up to CAP_MOST, a wider one (map_score).  At CAP_MOST the first form leaves a score 4.5e-5
// off, a hundredth of what rounding P to bf16 does; the wider form takes 628 us where it takes 503 (four rows of 2047, 16 heads over 4
// of 128, forward and backward).
constexpr int NO_CAP = 0, CAP = 1, WIDE_CAP = 2;
constexpr float CAP_MOST = 256.f;

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

// Walks the 64-row tiles first .. end - 1 that a workgroup's rows can share a document with.  `mine` / `whole`: whether the
// wave's own 32 rows meet the current tile, and whether every pair of the two is of one document.  Up or down: workgroups
// of a head that run at once should read the same tiles at once, so that they find them in their XCD's L2; queries (whose
// last tile differs) start at the front together, keys (whose first differs) at the end.
template <bool DOWN>
struct TileWalk {
    const int4* rg;                      // nullptr: no documents, every tile is visited whole
    int base, first, end;                // base: tiles behind us, in walking order
    DocRange block, wave;
    unsigned long long todo, mine_bits, whole_bits, pad_bits;
    bool mine, whole, pad;                // pad: some of the tile's rows are padding

    __device__ __forceinline__ void look(const int4& v) {          // v: this lane's entry (of a tile in range)
        bool a = base + (int)(threadIdx.x & 63) < end - first, b = true, c = true, p = false;
        if (rg != nullptr) {
            const DocRange d = merge(DocRange{v.x, v.y}, DocRange{v.z, v.w});
            a = a && meets(d, block);
            b = meets(d, wave);
            c = same_doc(d, wave);
            p = d.lo < 0;
        }
        todo = __ballot(a); mine_bits = __ballot(b); whole_bits = __ballot(c); pad_bits = __ballot(p);
    }
    __device__ __forceinline__ int tile(int n) const { return DOWN ? end - 1 - n : first + n; }
    __device__ __forceinline__ int4 entry() const {
        return rg != nullptr ? rg[tile(min(base + (int)(threadIdx.x & 63), end - first - 1))] : make_int4(0, 0, 0, 0);
    }
    // Rows row0 .. row0 + 127 (a multiple of 128; the wave's own are 32 w ..) against tiles first_ .. end_ - 1, end_ > first_.  One
    // round of loads: the entries of the rows' own two tiles and the first 64 of the walk go out together.
    __device__ __forceinline__ void open(const int4* rg_, int tiles, int row0, int w, int first_, int end_) {
        rg = rg_; base = 0; first = first_; end = end_;
        int4 v = entry();
        if (rg != nullptr) {
            const int t0 = row0 / TILE;
            const int4 o = rg[min(t0 + (int)(threadIdx.x & 1), tiles - 1)];
            const bool two = t0 + 1 < tiles;
            const auto lane_of = [](int x, int l) { return __builtin_amdgcn_readlane(x, l); };
            const int lo = min(o.x, o.z), hi = max(o.y, o.w), lo1 = lane_of(lo, 1), hi1 = lane_of(hi, 1);
            block = merge(DocRange{lane_of(lo, 0), lane_of(hi, 0)}, DocRange{two ? lo1 : 0x7fffffff, two ? hi1 : -0x7fffffff});
            const bool there = w < 2 || two;
            const int wlo = lane_of((w & 1) ? o.z : o.x, w >> 1), whi = lane_of((w & 1) ? o.w : o.y, w >> 1);
            wave = {there ? wlo : 0x7fffffff, there ? whi : -0x7fffffff};
        }
        look(v);
    }
    __device__ __forceinline__ void restart() { base = 0; look(entry()); }
    // the next tile, or `end` when there is none
    __device__ __forceinline__ int next() {
        while (todo == 0) {
            base += 64;
            if (base >= end - first) { base = end - first; return end; }
            look(entry());
        }
        const int bit = __ffsll((long long)todo) - 1;
        todo &= todo - 1;
        mine = (mine_bits >> bit) & 1; whole = (whole_bits >> bit) & 1; pad = (pad_bits >> bit) & 1;
        return tile(base + bit);
    }
};

// 64 rows x DH columns from memory straight into an LDS image (img_off), 16 bytes a lane and no registers in between: a wave's
// instruction fills 1 KiB in lane order, so the image's swizzle goes into which 16 bytes of the row each lane asks for.
// Rows past the last one are past the end of the descriptor and arrive as zeros; columns past D repeat the last eight (the
// other operand of every product that sums over them is zero there).  Completion: tiles_landed(), then a barrier.
template <int DH, int ROWS = TILE>
struct TileDma {
    const unsigned char* base;           // row 0
    unsigned step;                       // bytes of ROWS rows' strides
    unsigned whole, last;                // what a tile may read: a full one's bytes, the last one's
    unsigned off;                        // this lane's bytes in the tile's first rows
    // zeros: columns past D are zeros as well (for a tile whose partner's are not)
    __device__ __forceinline__ TileDma(const unsigned short* g, long rs, int T, int D, int tid, bool zeros = false) : base((const unsigned char*)g) {
        constexpr int CPR = DH / 8;
        const int row = tid / CPR, slot = tid % CPR;
        const int key = DH == 64 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
        const unsigned rb = (unsigned)rs * 2;
        off = row * rb + 2 * min((slot ^ key) * 8, D - 8);
        if (zeros && (slot ^ key) * 8 >= D) off = 0x80000000u;       // past any descriptor
        step = ROWS * rb;
        whole = (ROWS - 1) * rb + 2 * D;
        last = ((T - 1) % ROWS) * rb + 2 * D;
    }
    // rows ROWS j ..
    __device__ __forceinline__ void fetch(unsigned char* lds, int j, bool is_last, int wave) const {
        constexpr int LOADS = ROWS * DH * 2 / 4096;                  // of 256 / (DH / 8) rows each: a multiple of 16, so `key` repeats
        const u32x4 words = buffer_words(base + (unsigned long long)step * (unsigned)j, is_last ? last : whole);
        unsigned o = off;
        asm volatile("" : "+v"(o));                                  // the sums below are formed here, not kept across the loop
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            dma16<true>(__amdgpu_buffer_rsrc_t(), words, lds + i * 4096 + wave * 1024, o + i * (step / LOADS));
    }
};
// 64 words (documents, statistics) into LDS by one wave, a word a lane; zeros from word `n` on (all of them for n <= 0: a row's
// second 32 queries may not exist)
__device__ __forceinline__ void fetch_words(void* lds, const void* from, int n, int lane) {
    typedef __attribute__((address_space(3))) unsigned char* lds_byte_ptr;
    const unsigned at = (unsigned)(unsigned long long)(lds_byte_ptr)(unsigned char*)lds;
    const u32x4 words = buffer_words(from, (unsigned)__builtin_amdgcn_readfirstlane(min(max(n, 0), 64) * 4));
    dma_lds4(words, at, lane * 4);
}
// every load that this wave has issued is done
__device__ __forceinline__ void tiles_landed() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// rows of padding become zeros (docs: the tile's document numbers in LDS)
template <int DH, int ROWS = TILE>
__device__ __forceinline__ void clear_padding(unsigned char* lds, const int* docs, int tid) {
    constexpr int CPR = DH / 8, RSTEP = 256 / CPR;
    u32x4 zero = {0, 0, 0, 0};
    asm volatile("" : "+v"(zero));                                   // formed here, not kept across the loop
#pragma unroll
    for (int i = 0; i < ROWS * DH * 2 / 4096; ++i) {
        const int row = tid / CPR + i * RSTEP;
        if (docs[row] < 0) *(u32x4*)(lds + row * DH * 2 + (tid % CPR) * 16) = zero;
    }
}

// Where a lane reads its fragments in an image (img_off): the swizzle is an XOR of bits that lie below a row's size, so one
// offset per kind of read and an XOR with a constant give every fragment's place - 16 offsets kept in registers instead
// put the backward kernels past their budget.
template <int DH>
struct FragAt {
    unsigned row, tr;
    __device__ __forceinline__ explicit FragAt(int lane) {
        const int r = lane & 31, h = lane >> 5, tq = (lane & 15) >> 2, tp = lane & 3, gi = (lane >> 4) & 1;
        row = img_off<DH>(r, 8 * h);
        tr = img_off<DH>(4 * h + tq, 16 * gi + 4 * tp);
    }
    // the same in the image `base` bytes on (a multiple of a row).  The compiler takes the offsets for new ones: it forms the
    // XORs where they are used instead of keeping all of them in registers across the loop
    __device__ __forceinline__ FragAt at(unsigned base) const {
        FragAt f = *this;
        f.row += base; f.tr += base;
        asm volatile("" : "+v"(f.row), "+v"(f.tr));
        return f;
    }
    // A / B fragment kk of row 32 t2 + (lane & 31): elements 16 kk + 8 h ..;  img: bytes from the operand `base` names
    __device__ __forceinline__ bf16x8 rows(const unsigned char* smem, int img, int t2, int kk) const {
        return *(const bf16x8*)(smem + (row ^ (kk << 5)) + (img + 32 * t2 * DH * 2));
    }
    // transposed A fragment (tr_frag) of rows 32 t2 + 16 s + 4 h .., columns 32 di + (lane & 31)
    __device__ __forceinline__ bf16x8 cols(const unsigned char* smem, int img, int t2, int s, int di) const {
        const int k = img + (32 * t2 + 16 * s) * DH * 2;
        const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(smem + (tr ^ (di << 6)) + k));
        const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(smem + (tr ^ ((di << 6) | 32)) + (k + 8 * DH * 2)));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// this lane's half of one row as MFMA fragments, zero from column D on
template <int DH>
__device__ __forceinline__ void load_frags(const unsigned short* row, int h, int D, bf16x8 (&f)[DH / 16]) {
#pragma unroll
    for (int kk = 0; kk < DH / 16; ++kk) {
        const int col = 16 * kk + 8 * h;
        u32x4 v = {0, 0, 0, 0};
        if (col < D) v = *(const u32x4*)(row + col);
        f[kk] = __builtin_bit_cast(bf16x8, v);
    }
}
// ... and zero all over where the row is padding (apart from the loads: they need not wait for the document number)
template <int DH>
__device__ __forceinline__ void zero_unless(bool live, bf16x8 (&f)[DH / 16]) {
#pragma unroll
    for (int kk = 0; kk < DH / 16; ++kk) {
        const u32x4 v = __builtin_bit_cast(u32x4, f[kk]);
        f[kk] = __builtin_bit_cast(bf16x8, live ? v : u32x4{0, 0, 0, 0});
    }
}

template <int DI>
__device__ __forceinline__ void store_cols(unsigned short* __restrict__ dst, const floatx16 (&acc)[DI], float scale, int h, int D) {
#pragma unroll
    for (int di = 0; di < DI; ++di)
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

// A run of N matrix products fed from LDS: read(i) is issued AHEAD products in front of use(i, fragments).  Left to itself the
// compiler reads a fragment, waits for it and multiplies, one after the other.
// Here and in the other products a wave goes ahead of the SIMD's other waves: the matrix cores get the next product as soon as
// they can take it, and the others' vector work fills what is left (one row of 8192, 16 heads over 4: forward 358 -> 347 us,
// dQ 397 -> 367, dK / dV 525 -> 500; 16 heads of width 64: dK / dV 343 -> 330).
template <int N, int AHEAD, typename Read, typename Use>
__device__ __forceinline__ void feed(Read read, Use use) {
    __builtin_amdgcn_s_setprio(1);
    decltype(read(0)) f[AHEAD + 1];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i + AHEAD < N) f[(i + AHEAD) % (AHEAD + 1)] = read(i + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        use(i, f[i % (AHEAD + 1)]);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
}
struct Frag3 { bf16x8 a, b, c; };
struct Frag2 { bf16x8 a, b; };

// Scores in base 2 from raw products, and with a cap a quarter of 1 - tanh^2 in `f`.
//   CAP       r = 1 / (1 + e^{2u}), u = x / cap: cap (1 - 2 r), f = r (1 - r) with 1 - r as e^{2u} r: the difference itself has
//             nothing left where u < -8, and there f is all the gradient that a row of such scores has.
//   WIDE_CAP  relative accuracy wherever the score lies: below |u| = 0.4 the series of tanh(u) / u in u^2 (what is cut off is 4e-9),
//             from there on the same exponential of -2 |u|, which leaves 3e-7 of a tanh >= 0.38.
struct ScoreMap { float c, k1, cap2, k0; };   // scale log2 e;  2 scale log2 e / cap;  cap log2 e;  scale / cap
__device__ __forceinline__ ScoreMap score_map(const AttendArgs& a, int cap) {
    return {a.scale * LOG2E, cap ? 2.f * a.scale / a.softcap * LOG2E : 0.f, a.softcap * LOG2E, cap ? a.scale / a.softcap : 0.f};
}
template <int CAPPED>
__device__ __forceinline__ float map_score(const ScoreMap& m, float s, float& f) {
    if (CAPPED == CAP) {
        const float e = fast_exp2(s * m.k1), r = __builtin_amdgcn_rcpf(1.f + e);
        f = r * __builtin_amdgcn_fmed3f(e * r, 0.f, 1.f);           // (the clamp rides the product; an infinite e: r = 0, and the NaN of e r becomes 0)
        return fmaf(r, -2.f * m.cap2, m.cap2);
    }
    if (CAPPED == WIDE_CAP) {
        const float u = s * m.k0, w = u * u;
        float p = 21844.f / 6081075.f;
        p = fmaf(p, w, -1382.f / 155925.f);
        p = fmaf(p, w, 62.f / 2835.f);
        p = fmaf(p, w, -17.f / 315.f);
        p = fmaf(p, w, 2.f / 15.f);
        p = fmaf(p, w, -1.f / 3.f);
        p = fmaf(p, w, 1.f);
        const float t = u * p, e = fast_exp2(-fabsf(s * m.k1)), r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
        const bool near = w < 0.16f;
        f = near ? fmaf(-0.25f * t, t, 0.25f) : er * r;
        return near ? s * m.c * p : copysignf(fmaf(er, -2.f * m.cap2, m.cap2), s);
    }
    return s * m.c;
}

// In the query-stationary kernels the distance bias without a cap rides the score product as one more step of 16: rows (the 32 a fragment covers) bring their
// number in the tile, whole numbers up to 63 and so exact in bf16, columns bring their head's factor in three bf16 parts of 8
// bits each; the products are exact and their sum is fp32.  x = q . k + f row, in raw score units, leaves to the
// exponent's multiply-add a constant per lane and tile.  Right where |i - j| has one sign over the tile.
struct BiasFrag {
    unsigned row, f01, f2;               // 0 in the upper half of the wave, whose 8 elements of the step stay zero
    __device__ __forceinline__ BiasFrag(float f, int lane) {
        const __bf16 f0 = (__bf16)f, f1 = (__bf16)(f - (float)f0);
        row = lane < 32 ? float_to_bf16((float)lane) : 0u;
        f01 = lane < 32 ? pack_bf16x2(f, f - (float)f0) : 0u;
        f2 = lane < 32 ? float_to_bf16(f - (float)f0 - (float)f1) : 0u;
    }
    // rows 32 t2 ..: every row of the fragment 32 t2 on
    __device__ __forceinline__ floatx16 add(floatx16 S, int t2) const {
        unsigned r = t2 == 0 ? row : float_to_bf16(bf16_to_float((unsigned short)row) + 32.f), zero = 0;   // (the upper half's 32 meets zeros)
        asm volatile("" : "+v"(zero));   // formed here, not kept across the loop
        const u32x4 x = {r | (r << 16), r, zero, zero}, y = {f01, f2, zero, zero};
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), S, 0, 0, 0);
    }
};

// Masks shared by the kernels: how many keys at the front of a row every query sees (all of them without causality)
__device__ __forceinline__ int seen_prefix(const AttendArgs& a, int b) {
    if (!a.causal) return a.T;
    return a.prefix != nullptr ? min(max(a.prefix[b], 0), a.T) : 0;
}

// Which of a half tile's 32 rows a lane's column sees, as bits (row n: bit n), applied to the registers with a bit-field
// extract and a bitwise select: no lane masks in scalar registers, of which 16 comparisons would hold 32.
__device__ __forceinline__ unsigned range_bits(int from, int past) {              // rows from <= n < past
    const unsigned long long ones = 0xffffffffull;
    const unsigned lo = (unsigned)(ones << min(max(from, 0), 32)), hi = (unsigned)(ones >> (32 - min(max(past, 0), 32)));
    return lo & hi;
}
__device__ __forceinline__ unsigned doc_bits(const int* docs, int h, int mine) {  // rows acc_row(r, h) of the document `mine`; bit acc_row(r, 0)
    unsigned m = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) m |= docs[4 * h + acc_row(r, 0)] == mine ? 1u << acc_row(r, 0) : 0u;
    return mine >= 0 ? m : 0u;                                      // (padding sees no padding either)
}
__device__ __forceinline__ float pick(unsigned bits, int row, float x, float otherwise) {
    const int k = (int)(bits << (31 - row)) >> 31;
    const int xi = __builtin_bit_cast(int, x), oi = __builtin_bit_cast(int, otherwise);
    return __builtin_bit_cast(float, (xi & k) | (oi & ~k));
}

// Pipeline of the three kernels: two stages of LDS, each a 64-row tile of both streamed operands.  A stage's loads go out when
// the stage in front of it is about to be used and have that tile's products to arrive in; one barrier per tile says both
// that the tile is there and that nobody reads the stage that is filled next.
// (Three stages at width 64 changed nothing: 54 / 52 / 58 us on the short documents above.)
template <int DH> constexpr int stage_bytes() { return 2 * tile_bytes<DH>(); }
// waves per SIMD: what the registers of the accumulators and the stationary operand leave (512 / 2 at width 128)
template <int DH> constexpr int occupancy() { return DH == 64 ? 3 : 2; }

// ------------------------------------------------------------------------------ forward
template <int DH, int CAPPED, bool BIAS>
__global__ __launch_bounds__(256, occupancy<DH>()) void attend_fwd_kernel(AttendArgs a, unsigned short* __restrict__ out, unsigned short* __restrict__ rest, float* __restrict__ lse2) {
    constexpr int KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>(), SB = stage_bytes<DH>();
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SB];
    __shared__ __attribute__((aligned(256))) int Kds[2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 31, h = lane >> 5;
    const FragAt<DH> frags(lane);
    const int head = blockIdx.x, b = blockIdx.y, hk = head / (a.Hq / a.Hkv);
    const int T = a.T, q0 = (gridDim.z - 1 - blockIdx.z) * BQ, qw0 = q0 + 32 * wave, q = qw0 + ql, qc = min(q, T - 1);
    const unsigned short* qbase = (const unsigned short*)a.q + b * a.qb + head * a.qh;
    const TileDma<DH> kdma((const unsigned short*)a.k + b * a.kb + hk * a.kh, a.kt, T, a.D, tid);
    const TileDma<DH> vdma((const unsigned short*)a.v + b * a.vb + hk * a.vh, a.vt, T, a.D, tid);
    bf16x8 qf[KK];
    load_frags<DH>(qbase + (long)qc * a.qt, h, a.D, qf);
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = seen_prefix(a, b);
    const int lim = max(qc, pre - 1);                               // the last key that this lane's query sees
    const int qdoc = docs != nullptr ? docs[qc] : 0;
    const ScoreMap sm = score_map(a, CAPPED);
    const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
    const BiasFrag bf(BIAS && !CAPPED ? a.slopes[head] / a.scale : 0.f, lane);

    TileWalk<false> walk;
    walk.open(docs != nullptr ? a.ranges + (long)b * tiles : nullptr, tiles, q0, wave, 0, (max(min(q0 + BQ, T), pre) + TILE - 1) / TILE);
    const int wave_last = max(min(qw0 + 31, T - 1), pre - 1), wave_least = max(min(qw0, T - 1), pre - 1);

    int j = walk.next();
    if (j < walk.end) {
        kdma.fetch(smem, j, j == tiles - 1, wave);
        vdma.fetch(smem + TB, j, j == tiles - 1, wave);
        if (docs != nullptr && wave == 0) fetch_words(Kds[0], docs + j * TILE, T - j * TILE, lane);
    }
    zero_unless<DH>(qdoc >= 0, qf);
    floatx16 O[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) zero16(O[di]);
    float m = NEG_BIG, l = 0.f;
    for (int stage = 0; j < walk.end; stage ^= 1) {
        unsigned char* Ks = smem + stage * SB;
        unsigned char* Vs = Ks + TB;
        const int* Kd = Kds[stage];
        tiles_landed();
        __syncthreads();
        if (walk.pad) {                                             // workgroup-uniform
            clear_padding<DH>(Ks, Kd, tid);
            clear_padding<DH>(Vs, Kd, tid);
            __syncthreads();
        }
        const int jt = j * TILE;
        const bool go = walk.mine && jt <= wave_last, same = walk.whole, full = same && jt + TILE - 1 <= wave_least;
        j = walk.next();
        if (j < walk.end) {
            kdma.fetch(smem + (stage ^ 1) * SB, j, j == tiles - 1, wave);
            vdma.fetch(smem + (stage ^ 1) * SB + TB, j, j == tiles - 1, wave);
            if (docs != nullptr && wave == 0) fetch_words(Kds[stage ^ 1], docs + j * TILE, T - j * TILE, lane);
        }
        if (!go) continue;                                          // wave-uniform
        const FragAt<DH> fr = frags.at(stage * SB);
        floatx16 S[2];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            zero16(S[t2]);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                S[t2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.rows(smem, 0, t2, kk), qf[kk], S[t2], 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        // y = c S + add, in base 2: the scale and what is the same for a lane's whole tile ride the exponent's multiply-add
        float c = sm.c, add = 0.f;
        if (BIAS && !CAPPED && (jt + TILE - 1 <= qw0 || pre <= qw0)) {  // wave-uniform: no visible key lies behind its query
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) S[t2] = bf.add(S[t2], t2);
            add = slope2 * (float)(jt - q);
        } else if (CAPPED || BIAS) {
            c = 1.f;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float f;
                    S[t2][r] = map_score<CAPPED>(sm, S[t2][r], f);
                    if (BIAS) S[t2][r] = fmaf(-slope2, fabsf((float)(q - jt - 4 * h) - (float)(32 * t2 + acc_row(r, 0))), S[t2][r]);
                }
        }
        // Softmax and P V.  Tiles that are not seen whole hold the rows with few keys, whose O - and with it delta and all score
        // gradients - feels the rounding of single probabilities.  There the exponent is taken from the tile's own peak, so
        // that a row's only key has P = 1 exactly and leaves its V bit for bit, and what rounding P takes away goes through
        // the product as well.  (dK of 40-token documents is 2.5e-3 of its norm off without and 2.35e-3 with; where many keys
        // carry a row the errors average out.)  One body serves both products: accumulators that two paths leave are copied.
        if (!full) {                                                // wave-uniform
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                unsigned bits = range_bits(0, lim + 1 - jt - 32 * t2 - 4 * h);
                if (!same) bits &= doc_bits(Kd + 32 * t2, h, qdoc);
#pragma unroll
                for (int r = 0; r < 16; ++r) S[t2][r] = pick(bits, acc_row(r, 0), S[t2][r], MASKED);
            }
        }
        float mx = NEG_BIG;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[t2][r]);
        mx = xhalf_max(mx);
        const float peak = BIAS && !CAPPED ? fmaf(mx, c, add) : CAPPED ? mx : mx * c, mn = fmaxf(m, peak);
        const bool grew = mn > m;
        float off = BIAS && !CAPPED ? add - mn : -mn;
        if (!full) {
            off = peak >= m ? 0.f : peak - m;                       // (0 as such: the difference would be contracted)
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[t2][r] -= mx;
        }
        float rsum = 0.f;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = fast_exp2(CAPPED ? S[t2][r] + off : fmaf(S[t2][r], c, off));
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
        u32x4 pb[4], x[4];                                          // P as the product takes it, and what goes through it now
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pb[i] = __builtin_bit_cast(u32x4, pack_regs(S[i >> 1], i & 1));
        if (!full) {                                                // first what that rounding took
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8 f = __builtin_bit_cast(bf16x8, pb[i]);
                bf16x8 d;
#pragma unroll
                for (int k = 0; k < 8; ++k) d[k] = (__bf16)(S[i >> 1][8 * (i & 1) + k] - (float)f[k]);
                x[i] = __builtin_bit_cast(u32x4, d);
            }
        }
        __builtin_amdgcn_s_setprio(1);
        for (int pass = full ? 1 : 0; pass < 2; ++pass) {
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int di = 0; di < DI; ++di)
                        O[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.cols(smem, TB, t2, s, di), __builtin_bit_cast(bf16x8, x[2 * t2 + s]), O[di], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pb[i];
        }
        __builtin_amdgcn_s_setprio(0);
    }
    if (q < T) {
        const bool empty = l == 0.f;                                // saw no key: output zero, and P = exp2(x - 1e30) = 0 in backward
        const float inv = empty ? 0.f : 1.f / l;
        const long row = (((long)b * T + q) * a.Hq + head) * a.D;
#pragma unroll
        for (int di = 0; di < DI; ++di)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[di][r] *= inv;
        store_cols(out + row, O, 1.f, h, a.D);
        if (rest != nullptr) {
#pragma unroll
            for (int di = 0; di < DI; ++di)
#pragma unroll
                for (int r = 0; r < 16; ++r) O[di][r] -= bf16_to_float(float_to_bf16(O[di][r]));
            store_cols(rest + row, O, 1.f, h, a.D);
        }
        if (h == 0) lse2[((long)b * a.Hq + head) * T + q] = empty ? 1.0e30f : m + __log2f(l);
    }
}

// ------------------------------------------------------------------------------ dQ (query-stationary), and delta
template <int DH, int CAPPED, bool BIAS>
__global__ __launch_bounds__(256, occupancy<DH>()) void attend_bwd_q_kernel(AttendArgs a, const unsigned short* __restrict__ out, const unsigned short* __restrict__ rest,
                                                                            const unsigned short* __restrict__ dout, const float* __restrict__ lse2,
                                                                            float2* __restrict__ stats, unsigned short* __restrict__ dq) {
    constexpr int KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>(), SB = stage_bytes<DH>();
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SB];
    __shared__ __attribute__((aligned(256))) int Kds[2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 31, h = lane >> 5;
    const FragAt<DH> frags(lane);
    const int head = blockIdx.x, b = blockIdx.y, hk = head / (a.Hq / a.Hkv);
    const int T = a.T, q0 = (gridDim.z - 1 - blockIdx.z) * BQ, qw0 = q0 + 32 * wave, q = qw0 + ql, qc = min(q, T - 1);
    const unsigned short* qbase = (const unsigned short*)a.q + b * a.qb + head * a.qh;
    const TileDma<DH> kdma((const unsigned short*)a.k + b * a.kb + hk * a.kh, a.kt, T, a.D, tid);
    const TileDma<DH> vdma((const unsigned short*)a.v + b * a.vb + hk * a.vh, a.vt, T, a.D, tid);
    const long orow = (((long)b * T + qc) * a.Hq + head) * a.D;
    bf16x8 qf[KK], dof[KK];
    load_frags<DH>(qbase + (long)qc * a.qt, h, a.D, qf);
    load_frags<DH>(dout + orow, h, a.D, dof);
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = seen_prefix(a, b);
    const int lim = max(qc, pre - 1);
    const int qdoc = docs != nullptr ? docs[qc] : 0;
    const ScoreMap sm = score_map(a, CAPPED);
    const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
    const BiasFrag bf(BIAS && !CAPPED ? a.slopes[head] / a.scale : 0.f, lane);
    const float lse_q = lse2[((long)b * a.Hq + head) * T + qc];

    TileWalk<false> walk;
    walk.open(docs != nullptr ? a.ranges + (long)b * tiles : nullptr, tiles, q0, wave, 0, (max(min(q0 + BQ, T), pre) + TILE - 1) / TILE);
    const int wave_last = max(min(qw0 + 31, T - 1), pre - 1), wave_least = max(min(qw0, T - 1), pre - 1);
    int j = walk.next();
    if (j < walk.end) {
        kdma.fetch(smem, j, j == tiles - 1, wave);
        vdma.fetch(smem + TB, j, j == tiles - 1, wave);
        if (docs != nullptr && wave == 0) fetch_words(Kds[0], docs + j * TILE, T - j * TILE, lane);
    }

    float del;
    {
        bf16x8 of[KK], rf[KK];
        load_frags<DH>(out + orow, h, a.D, of);
        load_frags<DH>(rest + orow, h, a.D, rf);
        zero_unless<DH>(qdoc >= 0, qf);
        zero_unless<DH>(qdoc >= 0, dof);                            // out and rest of a padded row are zeros already
        floatx16 dd;
        zero16(dd);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) dd = __builtin_amdgcn_mfma_f32_32x32x16_bf16(of[kk], dof[kk], dd, 0, 0, 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) dd = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rf[kk], dof[kk], dd, 0, 0, 0);
        del = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) del = acc_row(r, h) == ql ? dd[r] : del;
        del = xhalf_sum(del);                                       // one half holds the diagonal element, the other zero
    }
    if (h == 0 && q < T) stats[((long)b * a.Hq + head) * T + q] = make_float2(BIAS ? fmaf(slope2, (float)(q % TILE), lse_q) : lse_q, del);

    floatx16 dQt[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) zero16(dQt[di]);
    for (int stage = 0; j < walk.end; stage ^= 1) {
        unsigned char* Ks = smem + stage * SB;
        unsigned char* Vs = Ks + TB;
        const int* Kd = Kds[stage];
        tiles_landed();
        __syncthreads();
        if (walk.pad) {
            clear_padding<DH>(Ks, Kd, tid);
            clear_padding<DH>(Vs, Kd, tid);
            __syncthreads();
        }
        const int jt = j * TILE;
        const bool go = walk.mine && jt <= wave_last, same = walk.whole;
        j = walk.next();
        if (j < walk.end) {
            kdma.fetch(smem + (stage ^ 1) * SB, j, j == tiles - 1, wave);
            vdma.fetch(smem + (stage ^ 1) * SB + TB, j, j == tiles - 1, wave);
            if (docs != nullptr && wave == 0) fetch_words(Kds[stage ^ 1], docs + j * TILE, T - j * TILE, lane);
        }
        if (!go) continue;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const int kt0 = jt + 32 * t2;
            if (kt0 > wave_last) continue;                          // wave-uniform
            const bool full = same && kt0 + 31 <= wave_least;
            const FragAt<DH> fr = frags.at(stage * SB);
            floatx16 S, dP;
            zero16(S); zero16(dP);
            feed<KK, 2>([&](int kk) { return Frag2{fr.rows(smem, 0, t2, kk), fr.rows(smem, TB, t2, kk)}; },
                        [&](int kk, const Frag2& f) {
                            S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a, qf[kk], S, 0, 0, 0);
                            dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.b, dof[kk], dP, 0, 0, 0);
                        });
            float c = sm.c, add = -lse_q;
            if (BIAS && !CAPPED && (kt0 + 31 <= qw0 || pre <= qw0)) {  // as in the forward
                S = bf.add(S, 0);
                add += slope2 * (float)(kt0 - q);
            } else if (BIAS && !CAPPED) {
                c = 1.f;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    S[r] = fmaf(S[r], sm.c, -slope2 * fabsf((float)(q - kt0 - 4 * h) - (float)acc_row(r, 0)));
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (CAPPED) {
                    float f, e = map_score<CAPPED>(sm, S[r], f);
                    if (BIAS) e = fmaf(-slope2, fabsf((float)(q - kt0 - 4 * h) - (float)acc_row(r, 0)), e);
                    S[r] = fast_exp2(e - lse_q) * (dP[r] - del) * f;                  // (1 - tanh^2) / 4; the rest behind the product
                } else {
                    S[r] = fast_exp2(fmaf(S[r], c, add)) * (dP[r] - del);
                }
            }
            if (!full) {
                unsigned bits = range_bits(0, lim + 1 - kt0 - 4 * h);
                if (!same) bits &= doc_bits(Kd + 32 * t2, h, qdoc);
#pragma unroll
                for (int r = 0; r < 16; ++r) S[r] = pick(bits, acc_row(r, 0), S[r], 0.f);
            }
            const bf16x8 dsb[2] = {pack_regs(S, 0), pack_regs(S, 1)};
            feed<2 * DI, 3>([&](int i) { return fr.cols(smem, 0, t2, i / DI, i % DI); },
                            [&](int i, bf16x8 f) { dQt[i % DI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, dsb[i / DI], dQt[i % DI], 0, 0, 0); });
        }
    }
    if (q < T) store_cols(dq + orow, dQt, qdoc >= 0 ? (CAPPED ? 4.f : 1.f) * a.scale : 0.f, h, a.D);
}

// ------------------------------------------------------------------------------ dK / dV (key-stationary, no atomics)
// A key head's gradient sums over its group of query heads.  Where that leaves few workgroups (kv_parts below) the group is
// cut: a workgroup takes `heads` of its query heads and writes its sums in fp32 to part [part][B, T, Hkv, D], dK and then dV,
// and fold_parts_kernel adds the parts in order.
// P and dS / scale (a quarter of it under a cap) of 32 queries (registers) and this lane's key, in place of S and dP.
// ld: the queries' (lse, delta) from row 4 h on; BIAS: lse + slope (i mod 64), so that -slope (i - j) - lse =
// slope (j - jt) - ld.x where no query that sees a key lies in front of it (`linear`), and elsewhere the sign is put right
// per element.  to_key: key - first query - 4 h; in_tile: key - first query of the 64-row tile.
template <int CAPPED, bool BIAS>
__device__ __forceinline__ void key_side(floatx16& S, floatx16& dP, const float2* ld, const ScoreMap& sm, float slope2, bool linear, int to_key, int in_tile) {
    const float add = slope2 * (float)in_tile, behind = !BIAS || linear ? 0.f : 2.f * slope2;
    if (BIAS && !CAPPED && !linear) {                                  // in raw units, in front of the scale
        const float f = behind / sm.c;
#pragma unroll
        for (int r = 0; r < 16; ++r) S[r] = fmaf(-f, fmaxf((float)to_key - (float)acc_row(r, 0), 0.f), S[r]);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = acc_row(r, 0);
        const float2 x = ld[row];
        float f, off = BIAS ? x.x - add : x.x;
        if (BIAS && CAPPED) off = fmaf(behind, fmaxf((float)to_key - (float)row, 0.f), off);
        S[r] = fast_exp2(CAPPED ? map_score<CAPPED>(sm, S[r], f) - off : fmaf(S[r], sm.c, -off));
        dP[r] = S[r] * (dP[r] - x.y);
        if (CAPPED) dP[r] *= f;                                     // (1 - tanh^2) / 4; the rest behind the product
    }
}

// this lane's key: rounded to dk / dv, or in fp32 to the workgroup's part (KvOut below)
struct KvOut {
    unsigned short *dk, *dv;
    float* part;                         // nullptr: whole groups
    int heads;                           // query heads of a workgroup
};
template <int CAPPED, int DI>
__device__ __forceinline__ void store_key(const AttendArgs& a, const KvOut& o, const floatx16 (&dKt)[DI], const floatx16 (&dVt)[DI], int b, int key, int hq0,
                                          bool live, int h) {
    if (key >= a.T) return;
    const int group = a.Hq / a.Hkv;
    const long row = (((long)b * a.T + key) * a.Hkv + hq0 / group) * a.D;
    const float kscale = live ? (CAPPED ? 4.f : 1.f) * a.scale : 0.f, vscale = live ? 1.f : 0.f;
    if (o.part == nullptr) {
        store_cols(o.dk + row, dKt, kscale, h, a.D);
        store_cols(o.dv + row, dVt, vscale, h, a.D);
        return;
    }
    const long n = (long)a.B * a.T * a.Hkv * a.D;
    float* to = o.part + (long)(hq0 % group / o.heads) * 2 * n + row;
#pragma unroll
    for (int di = 0; di < DI; ++di)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * di + 8 * g + 4 * h;
            if (d < a.D) {
                *(float4*)(to + d) = make_float4(dKt[di][4 * g] * kscale, dKt[di][4 * g + 1] * kscale, dKt[di][4 * g + 2] * kscale, dKt[di][4 * g + 3] * kscale);
                *(float4*)(to + n + d) = make_float4(dVt[di][4 * g] * vscale, dVt[di][4 * g + 1] * vscale, dVt[di][4 * g + 2] * vscale, dVt[di][4 * g + 3] * vscale);
            }
        }
}

template <int CAPPED, bool BIAS>
__global__ __launch_bounds__(256, 3) void attend_bwd_kv_kernel(AttendArgs a, const unsigned short* __restrict__ dout,
                                                               const float2* __restrict__ stats, KvOut o) {
    constexpr int DH = 64, KK = DH / 16, DI = DH / 32, TB = tile_bytes<DH>(), SB = stage_bytes<DH>();
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SB];
    __shared__ __attribute__((aligned(256))) float2 lds_ss[2][TILE];
    __shared__ __attribute__((aligned(256))) int Qds[2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kl = lane & 31, h = lane >> 5;
    const FragAt<DH> frags(lane);
    const int heads = o.heads, hq0 = blockIdx.x * heads, b = blockIdx.y, hk = hq0 / (a.Hq / a.Hkv);
    const int T = a.T, k0 = blockIdx.z * BQ, kw0 = k0 + 32 * wave, key = kw0 + kl, keyc = min(key, T - 1);
    const unsigned short* kbase = (const unsigned short*)a.k + b * a.kb + hk * a.kh;
    const unsigned short* vbase = (const unsigned short*)a.v + b * a.vb + hk * a.vh;
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int tiles = (T + TILE - 1) / TILE;
    const int pre = seen_prefix(a, b);
    const int kdoc = docs != nullptr ? docs[keyc] : 0;
    const ScoreMap sm = score_map(a, CAPPED);

    bf16x8 kf[KK], vf[KK];
    load_frags<DH>(kbase + (long)keyc * a.kt, h, a.D, kf);
    load_frags<DH>(vbase + (long)keyc * a.vt, h, a.D, vf);
    zero_unless<DH>(kdoc >= 0, kf);
    zero_unless<DH>(kdoc >= 0, vf);
    floatx16 dKt[DI], dVt[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) { zero16(dKt[di]); zero16(dVt[di]); }

    const int first = k0 < pre ? 0 : k0 / TILE;                     // in front of the first key only a prefix key is seen
    TileWalk<true> walk;
    walk.open(docs != nullptr ? a.ranges + (long)b * tiles : nullptr, tiles, k0, wave, first, tiles);
    const int key_from = key < pre ? -(1 << 30) : key;              // the first query that sees this lane's key

    for (int head = hq0; head < hq0 + heads; ++head) {
        const TileDma<DH> qdma((const unsigned short*)a.q + b * a.qb + head * a.qh, a.qt, T, a.D, tid);
        const TileDma<DH> odma(dout + ((long)b * T * a.Hq + head) * a.D, (long)a.Hq * a.D, T, a.D, tid);
        const float2* stats_b = stats + ((long)b * a.Hq + head) * T;
        const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
        if (head > hq0) walk.restart();
        int j = walk.next();
#define DPA_FETCH_Q(S_)                                                                                                  \
    if (j < walk.end) {                                                                                                  \
        qdma.fetch(smem + (S_) * SB, j, j == tiles - 1, wave);                                                                    \
        odma.fetch(smem + (S_) * SB + TB, j, j == tiles - 1, wave);                                                               \
        if (wave < 2) fetch_words(lds_ss[S_] + 32 * wave, stats_b + j * TILE + 32 * wave, 2 * (T - j * TILE - 32 * wave), lane);  \
        else if (wave == 2 && docs != nullptr) fetch_words(Qds[S_], docs + j * TILE, T - j * TILE, lane);                \
    }
        __syncthreads();                                            // the stages are free of the head before
        DPA_FETCH_Q(0)
        for (int stage = 0; j < walk.end; stage ^= 1) {
            unsigned char* Qs = smem + stage * SB;
            unsigned char* Os = Qs + TB;
            const float2* lds_s = lds_ss[stage];
            const int* Qd = Qds[stage];
            tiles_landed();
            __syncthreads();
            if (walk.pad) {
                clear_padding<DH>(Qs, Qd, tid);
                clear_padding<DH>(Os, Qd, tid);
                __syncthreads();
            }
            const int jt = j * TILE;
            const bool go = walk.mine && (jt + TILE - 1 >= kw0 || kw0 < pre), same = walk.whole;
            j = walk.next();
            DPA_FETCH_Q(stage ^ 1)
            if (!go) continue;                                      // wave-uniform
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const int qt0 = jt + 32 * t2;
                if (qt0 + 31 < kw0 && kw0 >= pre) continue;         // wave-uniform
                const bool full = same && (qt0 >= kw0 + 31 || kw0 + 31 < pre) && qt0 + 32 <= T;
                const FragAt<DH> fr = frags.at(stage * SB);
                floatx16 S, dP;
                zero16(S); zero16(dP);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.rows(smem, 0, t2, kk), kf[kk], S, 0, 0, 0);
                    dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.rows(smem, TB, t2, kk), vf[kk], dP, 0, 0, 0);
                }
                __builtin_amdgcn_s_setprio(0);
                const float2* ld4 = lds_s + 32 * t2 + 4 * h;
                key_side<CAPPED, BIAS>(S, dP, ld4, sm, slope2, qt0 >= kw0 + 31 || pre <= qt0, key - qt0 - 4 * h, key - jt);
                if (!full) {
                    unsigned bits = range_bits(key_from - qt0 - 4 * h, T - qt0 - 4 * h);
                    if (!same) bits &= doc_bits(Qd + 32 * t2, h, kdoc);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        S[r] = pick(bits, acc_row(r, 0), S[r], 0.f);
                        dP[r] = pick(bits, acc_row(r, 0), dP[r], 0.f);
                    }
                }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 pb = pack_regs(S, s), dsb = pack_regs(dP, s);
#pragma unroll
                    for (int di = 0; di < DI; ++di) {
                        dVt[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.cols(smem, TB, t2, s, di), pb, dVt[di], 0, 0, 0);
                        dKt[di] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.cols(smem, 0, t2, s, di), dsb, dKt[di], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
            }
        }
#undef DPA_FETCH_Q
    }
    store_key<CAPPED>(a, o, dKt, dVt, b, key, hq0, kdoc >= 0, h);
}

// The same at width 128.  Two accumulators of 32 keys x 128 channels and both stationary operands are 192 registers; with what
// two waves per SIMD leave beside them every fragment is read, waited for and used before the next one is read
// (one row of 8192, 16 heads over 4: 634 us, the form below 500).  So the workgroup's values stay in LDS instead, 32 KiB, and are read as they are needed; to fit two workgroups
// in a CU all the same, a stage is a half tile of 32 queries.
template <int CAPPED, bool BIAS>
__global__ __launch_bounds__(256, 2) void attend_bwd_kv_wide_kernel(AttendArgs a, const unsigned short* __restrict__ dout, const float2* __restrict__ stats, KvOut o) {
    constexpr int DH = 128, ROWS = 32, KK = DH / 16, DI = DH / 32, TB = ROWS * DH * 2, SB = 2 * TB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SB + BQ * DH * 2];   // two stages of queries and output gradients, then the values
    __shared__ __attribute__((aligned(256))) float2 lds_ss[2][TILE];      // (64 words land at once; the half's own are in front)
    __shared__ __attribute__((aligned(256))) int Qds[2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kl = lane & 31, h = lane >> 5;
    const FragAt<DH> frags(lane);
    const int heads = o.heads, hq0 = blockIdx.x * heads, b = blockIdx.y, hk = hq0 / (a.Hq / a.Hkv);
    const int T = a.T, k0 = blockIdx.z * BQ, kw0 = k0 + 32 * wave, key = kw0 + kl, keyc = min(key, T - 1);
    const int halves = (T + ROWS - 1) / ROWS, tiles = (T + TILE - 1) / TILE;
    {
        const TileDma<DH, ROWS> vdma((const unsigned short*)a.v + b * a.vb + hk * a.vh, a.vt, T, a.D, tid, true);
        for (int i = 0; i < BQ / ROWS; ++i)
            if (k0 / ROWS + i < halves) vdma.fetch(smem + 2 * SB + i * TB, k0 / ROWS + i, k0 / ROWS + i == halves - 1, wave);
    }
    bf16x8 kf[KK];
    load_frags<DH>((const unsigned short*)a.k + b * a.kb + hk * a.kh + (long)keyc * a.kt, h, a.D, kf);
    const int* docs = a.docs != nullptr ? a.docs + (long)b * T : nullptr;
    const int pre = seen_prefix(a, b);
    const int kdoc = docs != nullptr ? docs[keyc] : 0;
    const ScoreMap sm = score_map(a, CAPPED);
    zero_unless<DH>(kdoc >= 0, kf);                                 // (a padded key's values reach its own column of dP only, which its mask zeroes)
    floatx16 dKt[DI], dVt[DI];
#pragma unroll
    for (int di = 0; di < DI; ++di) { zero16(dKt[di]); zero16(dVt[di]); }
    TileWalk<true> walk;
    walk.open(docs != nullptr ? a.ranges + (long)b * tiles : nullptr, tiles, k0, wave, k0 < pre ? 0 : k0 / TILE, tiles);
    const int key_from = key < pre ? -(1 << 30) : key;

    for (int head = hq0; head < hq0 + heads; ++head) {
        const TileDma<DH, ROWS> qdma((const unsigned short*)a.q + b * a.qb + head * a.qh, a.qt, T, a.D, tid);
        const TileDma<DH, ROWS> odma(dout + ((long)b * T * a.Hq + head) * a.D, (long)a.Hq * a.D, T, a.D, tid);
        const float2* stats_b = stats + ((long)b * a.Hq + head) * T;
        const float slope2 = BIAS ? a.slopes[head] * LOG2E : 0.f;
        if (head > hq0) walk.restart();
        int n = 2 * walk.next();                                    // the half tile at hand; a tile's front half first
#define DPA_FETCH_Q(S_)                                                                                                  \
    if (n < halves) {                                                                                                    \
        qdma.fetch(smem + (S_) * SB, n, n == halves - 1, wave);                                                          \
        odma.fetch(smem + (S_) * SB + TB, n, n == halves - 1, wave);                                                     \
        if (wave == 0) fetch_words(lds_ss[S_], stats_b + n * ROWS, 2 * (T - n * ROWS), lane);                           \
        else if (wave == 1 && docs != nullptr) fetch_words(Qds[S_], docs + n * ROWS, T - n * ROWS, lane);                \
    }
        __syncthreads();                                            // the stages are free of the head before
        DPA_FETCH_Q(0)
        for (int stage = 0; n < halves; stage ^= 1) {
            tiles_landed();
            __syncthreads();
            if (walk.pad) {
                clear_padding<DH, ROWS>(smem + stage * SB, Qds[stage], tid);
                clear_padding<DH, ROWS>(smem + stage * SB + TB, Qds[stage], tid);
                __syncthreads();
            }
            const int qt0 = n * ROWS;
            const bool go = walk.mine && (qt0 + ROWS - 1 >= kw0 || kw0 < pre), same = walk.whole;
            n = (n & 1) == 0 && n + 1 < halves ? n + 1 : 2 * walk.next();
            DPA_FETCH_Q(stage ^ 1)
            if (!go) continue;                                      // wave-uniform
            const bool full = same && (qt0 >= kw0 + 31 || kw0 + 31 < pre) && qt0 + ROWS <= T;
            const FragAt<DH> fr = frags.at(stage * SB), fv = frags.at(2 * SB + wave * TB);
            floatx16 S, dP;
            zero16(S); zero16(dP);
            feed<KK, 2>([&](int kk) { return Frag3{fr.rows(smem, 0, 0, kk), fr.rows(smem, TB, 0, kk), fv.rows(smem, 0, 0, kk)}; },
                        [&](int kk, const Frag3& f) {
                            S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a, kf[kk], S, 0, 0, 0);
                            dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.b, f.c, dP, 0, 0, 0);
                        });
            key_side<CAPPED, BIAS>(S, dP, lds_ss[stage] + 4 * h, sm, slope2, qt0 >= kw0 + 31 || pre <= qt0, key - qt0 - 4 * h, key - qt0 / TILE * TILE);
            if (!full) {
                unsigned bits = range_bits(key_from - qt0 - 4 * h, T - qt0 - 4 * h);
                if (!same) bits &= doc_bits(Qds[stage], h, kdoc);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    S[r] = pick(bits, acc_row(r, 0), S[r], 0.f);
                    dP[r] = pick(bits, acc_row(r, 0), dP[r], 0.f);
                }
            }
            const bf16x8 pb[2] = {pack_regs(S, 0), pack_regs(S, 1)}, dsb[2] = {pack_regs(dP, 0), pack_regs(dP, 1)};
            feed<2 * DI, 2>([&](int i) { return Frag2{fr.cols(smem, TB, 0, i / DI, i % DI), fr.cols(smem, 0, 0, i / DI, i % DI)}; },
                            [&](int i, const Frag2& f) {
                                dVt[i % DI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a, pb[i / DI], dVt[i % DI], 0, 0, 0);
                                dKt[i % DI] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.b, dsb[i / DI], dKt[i % DI], 0, 0, 0);
                            });
        }
#undef DPA_FETCH_Q
    }
    tiles_landed();                                                 // where no query sees a key nobody has waited for the values
    store_key<CAPPED>(a, o, dKt, dVt, b, key, hq0, kdoc >= 0, h);
}

// dk, dv [n] = the sum of their parts [parts][2][n] in order, rounded once (n a multiple of 8)
__global__ __launch_bounds__(256) void fold_parts_kernel(const float* __restrict__ part, int parts, long n, unsigned short* __restrict__ dk,
                                                         unsigned short* __restrict__ dv) {
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < 2 * n; i += (long)gridDim.x * 256 * 8) {
        float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
        for (int p = 0; p < parts; ++p) {
            const float4 x = *(const float4*)(part + 2 * n * p + i), y = *(const float4*)(part + 2 * n * p + i + 4);
            s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w; s[4] += y.x; s[5] += y.y; s[6] += y.z; s[7] += y.w;
        }
        *(uint4*)(i < n ? dk + i : dv + i - n) = pack8(s);
    }
}

template <int DH, int CAPPED, bool BIAS>
void fwd_of(const AttendArgs& a, void* out, void* rest, float* lse2, hipStream_t st) {
    hipLaunchKernelGGL((attend_fwd_kernel<DH, CAPPED, BIAS>), dim3(a.Hq, a.B, (a.T + BQ - 1) / BQ), dim3(256), 0, st, a, (unsigned short*)out,
                       (unsigned short*)rest, lse2);
}
template <int DH, int CAPPED, bool BIAS>
void bwd_of(const AttendArgs& a, const void* out, const void* rest, const void* dout, const float* lse2, void* stats, void* dq, void* dk, void* dv,
            float* part, hipStream_t st) {
    const int blocks = (a.T + BQ - 1) / BQ;
    hipLaunchKernelGGL((attend_bwd_q_kernel<DH, CAPPED, BIAS>), dim3(a.Hq, a.B, blocks), dim3(256), 0, st, a, (const unsigned short*)out,
                       (const unsigned short*)rest, (const unsigned short*)dout, lse2, (float2*)stats, (unsigned short*)dq);
    const int parts = part != nullptr ? attend_kv_parts(a) : 1, heads = a.Hq / a.Hkv / parts;
    const KvOut o{(unsigned short*)dk, (unsigned short*)dv, part, heads};
    constexpr auto kv = DH == 64 ? attend_bwd_kv_kernel<CAPPED, BIAS> : attend_bwd_kv_wide_kernel<CAPPED, BIAS>;
    hipLaunchKernelGGL(kv, dim3(a.Hkv * parts, a.B, blocks), dim3(256), 0, st, a, (const unsigned short*)dout, (const float2*)stats, o);
    if (part != nullptr) {
        const long n = (long)a.B * a.T * a.Hkv * a.D, grid = (2 * n / 8 + 255) / 256;
        hipLaunchKernelGGL(fold_parts_kernel, dim3((unsigned)(grid > 8192 ? 8192 : grid)), dim3(256), 0, st, part, parts, n, (unsigned short*)dk, (unsigned short*)dv);
    }
}

}  // namespace

// one build per (width, cap, bias): the masks are wave-uniform branches inside
#define DPA_ATTEND_BIAS(F, DH_, CAP_, ...)                                                                              \
    do {                                                                                                                \
        if (a.slopes != nullptr) F<DH_, CAP_, true>(__VA_ARGS__); else F<DH_, CAP_, false>(__VA_ARGS__);                \
    } while (0)
#define DPA_ATTEND_CAP(F, DH_, ...)                                                                                     \
    do {                                                                                                                \
        if (!(a.softcap > 0.f)) DPA_ATTEND_BIAS(F, DH_, NO_CAP, __VA_ARGS__);                                           \
        else if (a.softcap <= CAP_MOST) DPA_ATTEND_BIAS(F, DH_, CAP, __VA_ARGS__);                                      \
        else DPA_ATTEND_BIAS(F, DH_, WIDE_CAP, __VA_ARGS__);                                                            \
    } while (0)
#define DPA_ATTEND_PICK(F, ...)                                                                                         \
    do {                                                                                                                \
        if (a.D <= 64) DPA_ATTEND_CAP(F, 64, __VA_ARGS__); else DPA_ATTEND_CAP(F, 128, __VA_ARGS__);                    \
    } while (0)

void attend_doc_ranges(const int* docs, void* ranges, int B, int T, hipStream_t st) {
    const int tiles = (T + TILE - 1) / TILE;
    hipLaunchKernelGGL(doc_ranges_kernel, dim3((tiles + 3) / 4, B), dim3(256), 0, st, docs, (int4*)ranges, T, tiles);
}

void attend_fwd(const AttendArgs& a, void* out, void* rest, float* lse2, hipStream_t st) { DPA_ATTEND_PICK(fwd_of, a, out, rest, lse2, st); }

// Query heads of a group in how many workgroups: the fewest that give 1024 of them (4 per CU: their work differs by where
// their keys stand), or one head each.  At width 128, 16 heads over 4, whole
// groups / 512 / 1024 workgroups took 1700 / 686 / 524 us on one row of 8192 and 565 / 249 / 220 on four of 2047
// (as it was when this was chosen); adding the parts
// takes 14 us for two and 23 for four.
int attend_kv_parts(const AttendArgs& a) {
    const int group = a.Hq / a.Hkv;
    const long wgs = (long)a.Hkv * a.B * ((a.T + BQ - 1) / BQ);
    for (int p = 1; p < group; ++p)
        if (group % p == 0 && wgs * p >= 1024) return p;
    return group;
}

void attend_bwd(const AttendArgs& a, const void* out, const void* rest, const void* dout, const float* lse2, void* stats, void* dq, void* dk, void* dv,
                float* part, hipStream_t st) {
    DPA_ATTEND_PICK(bwd_of, a, out, rest, dout, lse2, stats, dq, dk, dv, part, st);
}

}  // namespace dpa
