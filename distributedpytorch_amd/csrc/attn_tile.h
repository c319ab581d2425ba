// Pieces that the attention kernels (attention.hip, attend.hip) share: the LDS image of a 64-row tile, the MFMA
// fragments read from it, and the cross-half reductions of a wave.
#pragma once
#include "common.h"

namespace dpa {
namespace attn {

constexpr int TILE = 64;                 // rows per staged tile
constexpr float NEG_BIG = -1.0e30f;
template <int DH> constexpr int tile_bytes() { return TILE * DH * 2; }   // 8 / 16 KiB

typedef __attribute__((address_space(3))) short4v* lds_s4_ptr;

// byte offset of element (row, col) in a [64][DH] bf16 LDS image that serves row reads (ds_read_b128) and transposed
// reads (ds_read_b64_tr_b16) alike.  DH = 64 (128-byte rows, two rows per 256-byte bank row): the 16-byte chunk index
// XORed with (bit 1 of the row) << 2 | (row >> 2) & 3.  Bit 2 of the key moves rows 4m+2, 4m+3 to the other 64-byte
// window than rows 4m, 4m+1, so the 4 rows x 64 bytes of a transposed read cover the bank row once; the low bits make
// the 8 same-parity rows of a ds_read_b128 lane group ({0-3, 12-15, 20-27} / {4-11, 16-19, 28-31}) use 8 different
// chunks.  (A 64-byte-granule swizzle served the transposed reads only: PMC showed the row reads 4-way conflicted,
// 45-59 % of the three kernels' LDS cycles - profiles/pmc/attn_*.txt.)  DH = 128 (256-byte rows): the chunk index
// XORed with ((row & 3) << 2 | (row >> 2) & 3) - conflict-free for both kinds of read.
template <int DH>
__device__ __forceinline__ int img_off(int row, int col) {
    if (DH == 64) return row * 128 + ((((col >> 3) ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3))) & 7) << 4) + (col & 7) * 2;
    return row * 256 + ((((col >> 3) ^ (((row & 3) << 2) | ((row >> 2) & 3))) & 15) << 4) + (col & 7) * 2;
}

// Global loads of a 64 x DH bf16 tile (row stride `rs` elements, first row `r0`, rows clamped to `rlast`) split in
// two, so the next tile's loads are in flight under the current tile's MFMAs: fetch_tile issues them into registers,
// stash_tile writes the registers to the LDS image
template <int DH>
__device__ __forceinline__ void fetch_tile(const unsigned short* __restrict__ g, long rs, int r0, int rlast, int tid,
                                           u32x4 (&r)[DH / 32]) {
    constexpr int CPR = DH / 8, RSTEP = 256 / CPR;
    const int c = tid % CPR;
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) {
        int row = r0 + tid / CPR + i * RSTEP;
        row = row < rlast ? row : rlast;
        r[i] = *(const u32x4*)(g + (long)row * rs + c * 8);
    }
}
template <int DH>
__device__ __forceinline__ void stash_tile(unsigned char* lds, int tid, const u32x4 (&r)[DH / 32]) {
    constexpr int CPR = DH / 8, RSTEP = 256 / CPR;
    const int c = tid % CPR;
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) *(u32x4*)(lds + img_off<DH>(tid / CPR + i * RSTEP, c * 8)) = r[i];
}

// MFMA A/B row fragment: 8 consecutive d of one row (k = 8h + j + 16kk)
template <int DH>
__device__ __forceinline__ bf16x8 row_frag(const unsigned char* lds, int row, int kk, int h) {
    return *(const bf16x8*)(lds + img_off<DH>(row, 16 * kk + 8 * h));
}

// transposed A fragment for  Y^T[d][..] += T^T[d x rows] . X[rows x ..]  where X is an
// accumulator tile used as B operand: element j <-> row rowbase + 8(j>>2) + (j&3)
// (rowbase already contains 16s + 4h), d = dbase + (lane & 31)
template <int DH>
__device__ __forceinline__ bf16x8 tr_frag(const unsigned char* lds, int rowbase, int dbase, int lane) {
    const int gi = lane >> 4, li = lane & 15, tq = li >> 2, tp = li & 3;
    const int col = dbase + (gi & 1) * 16 + 4 * tp;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(lds + img_off<DH>(rowbase + tq, col)));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(lds + img_off<DH>(rowbase + 8 + tq, col)));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ bf16x8 pack_regs(const floatx16& x, int s) {   // registers 8s .. 8s+7 -> bf16x8
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (__bf16)x[8 * s + j];
    return r;
}

// 2^x as ONE v_exp_f32: arguments here are <= 0 (score minus running max / log-sum-exp), so exp2f's denormal
// and overflow range handling (5 extra VALU instructions per element) buys nothing; very negative -> 0.
typedef float float2v __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The two halves of a wave hold the two halves of a query's row statistics: combine lane i with lane i ^ 32 through
// gfx950's v_permlane32_swap (a vector-ALU instruction) instead of __shfl_xor's ds_bpermute, which is an LDS round trip
// with a wait in the middle of every tile's dependency chain.  swap(x, x) returns (low half twice, high half twice).
// (The results are copied into scalars before the bit cast: __builtin_bit_cast applied to `r[1]` itself reads element 0 with
// this compiler - the sum came out as 2 * r[0].)
__device__ __forceinline__ void xhalf_swap(float x, float& lo, float& hi) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const u32x2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r.x, b = r.y;
    lo = __builtin_bit_cast(float, a);
    hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float xhalf_max(float x) {
    float lo, hi;
    xhalf_swap(x, lo, hi);
    return fmaxf(lo, hi);
}
__device__ __forceinline__ float xhalf_sum(float x) {
    float lo, hi;
    xhalf_swap(x, lo, hi);
    return lo + hi;
}

__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

__device__ __forceinline__ void zero16(floatx16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}

// store transposed accumulators (rows = d, col = this lane's token) as bf16 [token][DH]
template <int DH>
__device__ __forceinline__ void store_T(unsigned short* __restrict__ dst, const floatx16 (&acc)[DH / 32], float scale, int h) {
#pragma unroll
    for (int di = 0; di < DH / 32; ++di)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * di + 8 * g + 4 * h;
            uint2 pk;
            pk.x = pack_bf16x2(acc[di][4 * g + 0] * scale, acc[di][4 * g + 1] * scale);
            pk.y = pack_bf16x2(acc[di][4 * g + 2] * scale, acc[di][4 * g + 3] * scale);
            *(uint2*)(dst + d) = pk;
        }
}

}  // namespace attn
}  // namespace dpa
