// Token embedding with a scale, and its gradient by sorted tokens (gfx950).
//
//   y[i] = scale * W[tok_i];    dW[v] = scale * sum over { i : tok_i = v } of dy[i], positions ascending.
//   An id outside [0, V) names no row: its output row is zero and it adds to no gradient.
//
// Bound by memory: the forward reads a table row per token and writes one; the backward reads dy once and writes dW once.
// Backward in two launches (three from 512 tokens on), no atomics, every sum in one fixed order:
//   1. sort_tokens: a workgroup owns every 256th run of 8 ids (vocabularies put their common words side by side, and a range
//      of ids would be one workgroup's work; single ids would leave the rows' sums no neighbours to share cache lines with).
//      It reads the whole token list, counts its ids - and the tokens that groups before it own, which is where its output
//      begins, so that no workgroup waits for another - and notes where they stand.  Each of its 16 waves owns a contiguous
//      piece of the list and a histogram of its own; the histograms summed over waves and ids give every (wave, id) its
//      place, and inside a wave equal ids are ranked by ballots, so the sort is stable.  Reading the list in every workgroup
//      costs L2 traffic only; a sort by passes over digits would cost two launches a digit.  65,536 tokens over 50,304 ids:
//      24 us, 39 with the common ids side by side (with ranges of ids, and the list read again to place them: 35 and 268).
//   2. sum_runs: the sorted list in chunks of 64; what a chunk holds of one id is summed to a partial row where that is 16
//      tokens or more.  This is where frequent tokens (6 % of a text are its commonest one) are spread over the chip.
//   3. sum_rows: a thread per 8 channels of every table row adds the row's entries - long runs through their partials - and
//      writes the row, zeros where no token named it: the gradient needs no clearing beforehand.
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

constexpr int SORT_WAVES = 16, BATCH = 16, CHUNK = 64, LONG = 16;
constexpr int SIDE_BITS = 3;                  // ids that stay side by side: 2^3
constexpr int OWN_BITS = 9, HELD = 448;       // ids of a workgroup at most 2^9; places that a wave notes: 28 KiB beside 32 of counters

template <typename I>
__global__ __launch_bounds__(256) void token_embedding_fwd_kernel(const I* __restrict__ tok, const unsigned short* __restrict__ w, unsigned short* __restrict__ y,
                                                                  long n, int C, long V, float scale) {
    const int nch = C / 8, rows = nch >= 256 ? 1 : 256 / nch;
    for (long r0 = (long)blockIdx.x * rows; r0 < n; r0 += (long)gridDim.x * rows)
    for (int i = threadIdx.x; i < rows * nch; i += 256) {
        const int dr = i / nch, ch = i - dr * nch;
        const long row = r0 + dr;
        if (row >= n) break;
        const long id = (long)tok[row];
        float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (id >= 0 && id < V) {
            const uint4 u = *(const uint4*)(w + id * C + ch * 8);
            unpack8(u, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= scale;
        }
        *(uint4*)(y + row * C + ch * 8) = pack8(f);
    }
}

// order[]: positions sorted by (group, id, position), sorted[]: what stands there; span[v]: id v's part of it, span[V].x: how
// many tokens there are.  Workgroup b of 2^g owns the ids whose g bits above the last SIDE_BITS are b, at most `width`; LDS: SORT_WAVES * width counters.
template <typename I>
__global__ __launch_bounds__(64 * SORT_WAVES) void sort_tokens_kernel(const I* __restrict__ tok, int n, unsigned V, int g, int width,
                                                                      int2* __restrict__ span, int* __restrict__ order, int* __restrict__ sorted) {
    extern __shared__ int hist[];                         // [SORT_WAVES][width]
    __shared__ unsigned held[SORT_WAVES][HELD];           // (place in the wave's piece) << 9 | own id
    __shared__ int below_s[SORT_WAVES], scan_s[SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // ids turned right by g + SIDE_BITS: the group on top, so that one comparison each finds the groups before and its own
    const unsigned lo = blockIdx.x << (32 - g), last = lo + ((1u << (32 - g)) - 1);
    for (int i = tid; i < SORT_WAVES * width; i += 64 * SORT_WAVES) hist[i] = 0;
    __syncthreads();
    const int piece = ((n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
    const int p0 = wave * piece, p1 = p0 + piece < n ? p0 + piece : n;
    int below = 0, cnt = 0, resume = 0;                   // tokens noted; the first that no longer was
    int* mine = hist + wave * width;
    // Tokens from `from` on: 64 x BATCH at a time, all loads of a batch on their way before the first is looked at - one after
    // the other they are a chain of L2 round trips (16,384 tokens: 18 us against 11).
    const auto scan = [&](int from, bool count) {
        cnt = 0;
        resume = p1;
        for (int p = from; p < p1 && (count || resume == p1); p += 64 * BATCH) {
            I t[BATCH];
            if (p + 64 * BATCH <= p1) {                   // wave-uniform: no test per token
#pragma unroll
                for (int i = 0; i < BATCH; ++i) t[i] = tok[p + 64 * i + lane];
            } else {
#pragma unroll
                for (int i = 0; i < BATCH; ++i) t[i] = p + 64 * i + lane < p1 ? tok[p + 64 * i + lane] : (I)-1;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const bool there = sizeof(I) == 8 ? (unsigned long long)t[i] < V : (unsigned)t[i] < V;
                const unsigned x = __builtin_rotateright32((unsigned)t[i], (unsigned)(g + SIDE_BITS));
                const bool hit = there && x >= lo && x <= last;
                const unsigned long long hits = __ballot(hit);
                if (count) below += __popcll(__ballot(there && x < lo));
                if (hits == 0) continue;                  // wave-uniform
                const unsigned v = ((unsigned)t[i] >> (g + SIDE_BITS) << SIDE_BITS) | ((unsigned)t[i] & ((1u << SIDE_BITS) - 1));
                if (count && hit) atomicAdd(&mine[v], 1);
                if (resume < p1) continue;
                if (cnt + __popcll(hits) > HELD) { resume = p + 64 * i; continue; }
                if (hit) held[wave][cnt + __popcll(hits & ((1ull << lane) - 1))] = ((unsigned)(p - p0 + 64 * i + lane) << OWN_BITS) | v;
                cnt += __popcll(hits);
            }
        }
    };
    scan(p0, true);
    if (lane == 0) below_s[wave] = below;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) base += below_s[w];
    // exclusive scan of the ids' totals (at most 2^9); each (wave, id) counter becomes its first place
    const unsigned id = ((unsigned)tid >> SIDE_BITS << (g + SIDE_BITS)) | (blockIdx.x << SIDE_BITS) | (tid & ((1u << SIDE_BITS) - 1));
    const bool owned = tid < width && id < V;
    int total = 0;
    if (owned)
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) total += hist[w * width + tid];
    int inc = total;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int t = __shfl_up(inc, off, 64);
        if (lane >= off) inc += t;
    }
    if (lane == 63) scan_s[wave] = inc;
    __syncthreads();
    int at = base + inc - total;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) at += w < wave ? scan_s[w] : 0;
    if (owned) {
        span[id] = make_int2(at, at + total);
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int c = hist[w * width + tid];
            hist[w * width + tid] = at;
            at += c;
        }
    }
    if (blockIdx.x == gridDim.x - 1 && tid == 64 * SORT_WAVES - 1) span[V].x = at;      // (nothing is left to add there)
    __syncthreads();
    for (;;) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i0 = 0; i0 < cnt; i0 += 64) {
            const bool hit = i0 + lane < cnt;
            const unsigned e = hit ? held[wave][i0 + lane] : 0u, v = e & ((1u << OWN_BITS) - 1);
            int rank = 0, same_ids = 0;
            unsigned long long left = __ballot(hit);
            while (left != 0) {                           // one distinct id per turn
                const unsigned u = __builtin_amdgcn_readlane(v, __ffsll((long long)left) - 1);
                const unsigned long long same = __ballot(hit && v == u);
                if (v == u) { rank = __popcll(same & ((1ull << lane) - 1)); same_ids = __popcll(same); }
                left &= ~same;
            }
            const int first = mine[v];
            if (hit) {
                order[first + rank] = p0 + (int)(e >> OWN_BITS);
                sorted[first + rank] = (int)((v << g) | blockIdx.x);         // (told apart is all that they need)
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (hit && rank == same_ids - 1) mine[v] = first + same_ids;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (resume >= p1) break;
        scan(resume, false);
    }
}

// The sorted list in chunks of 64.  What a chunk holds of one id is a run; the runs of at least LONG tokens - at most
// CHUNK / LONG to a chunk, told apart by which LONG of the chunk they begin in - are summed to partial rows of their own.
__device__ __forceinline__ long partial_row(int first) { return first / LONG; }

// partial[partial_row(first)][C] = sum of the run's rows
__global__ __launch_bounds__(256) void sum_runs_kernel(const int* __restrict__ order, const int* __restrict__ sorted, const int2* __restrict__ span,
                                                       long V, const unsigned short* __restrict__ dy, float* __restrict__ partial, int C) {
    __shared__ float red[4][64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = blockIdx.x * CHUNK, n = min(span[V].x - s, CHUNK);
    if (n < LONG) return;
    const int id = sorted[s + min(lane, n - 1)], before = __shfl_up(id, 1, 64);
    const unsigned long long heads = __ballot(lane == 0 || id != before) & (~0ull >> (64 - n));
    const int nch = C / 8;
    for (unsigned long long left = heads; left != 0; left &= left - 1) {
        const int a = __ffsll((long long)left) - 1;
        const unsigned long long rest = left & (left - 1);
        const int b = rest != 0 ? __ffsll((long long)rest) - 1 : n;
        if (b - a < LONG) continue;
        for (int c0 = 0; c0 < nch; c0 += 64) {
            const int ch = c0 + lane;
            float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (ch < nch) {
#pragma unroll 4
                for (int i = a + wave; i < b; i += 4) {
                    float f[8];
                    const uint4 u = *(const uint4*)(dy + (long)order[s + i] * C + ch * 8);
                    unpack8(u, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[j] += f[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) red[wave][lane * 8 + j] = acc[j];
            __syncthreads();
            for (int i = threadIdx.x; i < 512; i += 256)
                if (c0 * 8 + i < C) partial[partial_row(s + a) * C + c0 * 8 + i] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
            __syncthreads();
        }
    }
}

__device__ __forceinline__ floatx4 four(const unsigned short* p) {
    const uint2 u = *(const uint2*)p;
    return floatx4{bf16_to_float(u.x & 0xffff), bf16_to_float(u.x >> 16), bf16_to_float(u.y & 0xffff), bf16_to_float(u.y >> 16)};
}
__device__ __forceinline__ void add_rows(floatx4 (&acc)[2], const int* __restrict__ order, int s, int e, const unsigned short* __restrict__ dy, int C, int c) {
#pragma unroll 4
    for (int i = s; i < e; ++i) {
        const unsigned short* p = dy + (long)order[i] * C + c;
        acc[0] += four(p);
        acc[1] += four(p + C / 2);
    }
}

__device__ __forceinline__ void add_partial(floatx4 (&acc)[2], const float* __restrict__ partial, int first, int C, int c) {
    const float* p = partial + partial_row(first) * C + c;
    acc[0] += *(const floatx4*)p;
    acc[1] += *(const floatx4*)(p + C / 2);
}

// A thread has four channels in each half of the row: as many loads in flight as with eight together, and stores that leave no
// gaps between lanes.  The rows are stored past the caches, which they would only fill (16,384 tokens over 50,304 x 768, inputs not
// in cache: 65 us with both otherwise, 40 so, and 31 since no row waits for more than LONG - 1 single entries on either side;
// storing the zeros of 50,304 x 768 alone takes 23).  Eight loads at once instead of four cost the waves that hide them (65,536
// tokens: 104 against 89 us).
// ADD: rows that some token names are added to dw (which another stream may be adding to as well: one atomic per element);
// otherwise every row is written
template <bool ADD>
__global__ __launch_bounds__(256) void sum_rows_kernel(const int* __restrict__ order, const int2* __restrict__ span, const unsigned short* __restrict__ dy,
                                                       const float* __restrict__ partial, float* __restrict__ dw, long V, int C, float scale, int rows) {
    // a workgroup takes `rows` rows: only the place within them is divided, in 32 bits
    const int nch = C / 8;
    const long v0 = (long)blockIdx.x * rows;
    for (int i = threadIdx.x; i < rows * nch; i += 256) {
        const int dv = i / nch, c = (i - dv * nch) * 4;
        const long v = v0 + dv;
        if (v >= V) break;
        const int s = span[v].x, e = span[v].y;
        floatx4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        // the run in the first chunk, whole chunks, the run in the last one
        const int first = partial != nullptr ? min(e, (s / CHUNK + 1) * CHUNK) : s, last = max(first, e / CHUNK * CHUNK);
        int from = s;
        if (first - s >= LONG) {
            add_partial(acc, partial, s, C, c);
            from = first;
        }
        const int mid = partial != nullptr ? first : e;
        add_rows(acc, order, from, mid, dy, C, c);
        if (partial != nullptr) {
#pragma unroll 4
            for (int k = first; k < last; k += CHUNK) add_partial(acc, partial, k, C, c);
            if (e - last >= LONG) add_partial(acc, partial, last, C, c);
            else add_rows(acc, order, last, e, dy, C, c);
        }
        acc[0] *= scale;
        acc[1] *= scale;
        float* o = dw + v * C + c;
        if (ADD) {
            if (s < e)
#pragma unroll
                for (int j = 0; j < 8; ++j) unsafeAtomicAdd(o + (j & 3) + (j >> 2) * (C / 2), acc[j >> 2][j & 3]);
        } else {
            __builtin_nontemporal_store(acc[0], (floatx4*)o);
            __builtin_nontemporal_store(acc[1], (floatx4*)(o + C / 2));
        }
    }
}

inline unsigned blocks_for(long threads, long cap) {
    long b = (threads + 255) / 256;
    return (unsigned)(b < 1 ? 1 : b > cap ? cap : b);
}

// the most ids that a workgroup of 2^g has
inline int sort_width(long V, int g) { return (int)((((V - 1) >> (g + SIDE_BITS)) + 1) << SIDE_BITS); }
// workgroups of the sort as a power of two: 256, one to a CU, or as many as leave each 2^9 ids
inline int sort_bits(long V) {
    int g = 1;
    while (((1l << SIDE_BITS) << g) < V && (g < 8 || sort_width(V, g) > (1 << OWN_BITS))) ++g;
    return g;
}

template <typename I>
void backward_of(const I* tok, const void* dy, float* dw, int add, long n, int C, long V, float scale, int2* span, int* order, int* sorted,
                 float* partial, hipStream_t st) {
    const int g = sort_bits(V), width = sort_width(V, g);
    hipLaunchKernelGGL((sort_tokens_kernel<I>), dim3(1u << g), dim3(64 * SORT_WAVES), SORT_WAVES * width * sizeof(int), st,
                       tok, (int)n, (unsigned)V, g, width, span, order, sorted);
    if (partial != nullptr)
        hipLaunchKernelGGL(sum_runs_kernel, dim3((unsigned)((n + CHUNK - 1) / CHUNK)), dim3(256), 0, st, order, sorted, span, V, (const unsigned short*)dy, partial, C);
    const int rows = C / 8 >= 512 ? 1 : 512 / (C / 8);
    const dim3 blocks((unsigned)((V + rows - 1) / rows));
    if (add)
        hipLaunchKernelGGL((sum_rows_kernel<true>), blocks, dim3(256), 0, st, order, span, (const unsigned short*)dy, partial, dw, V, C, scale, rows);
    else
        hipLaunchKernelGGL((sum_rows_kernel<false>), blocks, dim3(256), 0, st, order, span, (const unsigned short*)dy, partial, dw, V, C, scale, rows);
}

}  // namespace

void token_embedding_fwd(const void* tok, int tok64, const void* w, void* y, long n, int C, long V, float scale, hipStream_t st) {
    if (n == 0) return;
    const long rows = C / 8 >= 256 ? 1 : 256 / (C / 8);
    const unsigned blocks = blocks_for((n + rows - 1) / rows * 256, 1 << 20);
    if (tok64)
        hipLaunchKernelGGL((token_embedding_fwd_kernel<int64_t>), dim3(blocks), dim3(256), 0, st, (const int64_t*)tok, (const unsigned short*)w, (unsigned short*)y, n, C, V, scale);
    else
        hipLaunchKernelGGL((token_embedding_fwd_kernel<int>), dim3(blocks), dim3(256), 0, st, (const int*)tok, (const unsigned short*)w, (unsigned short*)y, n, C, V, scale);
}

long token_embedding_partials(long n) { return n >= 8 * CHUNK ? (n + LONG - 1) / LONG : 0; }

void token_embedding_bwd(const void* tok, int tok64, const void* dy, float* dw, int add, long n, int C, long V, float scale, void* span, int* order,
                         int* sorted, float* partial, hipStream_t st) {
    if (tok64) backward_of((const int64_t*)tok, dy, dw, add, n, C, V, scale, (int2*)span, order, sorted, partial, st);
    else backward_of((const int*)tok, dy, dw, add, n, C, V, scale, (int2*)span, order, sorted, partial, st);
}

}  // namespace dpa
