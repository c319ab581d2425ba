// Token embedding with a scale, and its gradient by sorted tokens (gfx950).
//
//   y[i] = scale * W[tok_i];    dW[v] = scale * sum over { i : tok_i = v } of dy[i], positions ascending.
//   An id outside [0, V) names no row: its output row is zero and it adds to no gradient.
//
// Bound by memory: the forward reads a table row per token and writes one; the backward reads dy once and writes dW once.
// Backward in two launches (three from 512 tokens on), no atomics, every sum in one fixed order:
//   1. sort_tokens: a workgroup owns a range of ids.  It reads the whole token list twice - once to count its ids (and the
//      tokens below its range, which is where its output begins, so that no workgroup waits for another), once to place
//      them.  Each of its 16 waves owns a contiguous piece of the list and a histogram of its own; the histograms summed
//      over waves and ids give every (wave, id) its place, and inside a wave equal ids are ranked by ballots, so the sort
//      is stable.  Re-reading the list costs L2 traffic only; a sort by passes over digits would cost two launches a digit.
//   2. sum_chunks: the sorted list in chunks of 64; a chunk that lies inside ONE id's segment is summed to a partial row.
//      This is where frequent tokens (6 % of a text are its commonest one) are spread over the chip.
//   3. sum_rows: a thread per 8 channels of every table row adds the row's entries - whole chunks through their partials - and
//      writes the row, zeros where no token named it: the gradient needs no clearing beforehand.
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

constexpr int SORT_WAVES = 16, BATCH = 16, CHUNK = 64;

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

// an id as 32 bits, -1 for one that no table of fewer than 2^31 rows has
__device__ __forceinline__ int small_id(int id) { return id; }
__device__ __forceinline__ int small_id(int64_t id) { return (unsigned long long)id < 0x7fffffffull ? (int)id : -1; }

// order[]: positions sorted by (id, position); start[v] .. start[v + 1]: id v's part of it.  Workgroup b owns ids
// [b * width, min(V, (b + 1) * width)); LDS: SORT_WAVES * width counters.
template <typename I>
__global__ __launch_bounds__(64 * SORT_WAVES) void sort_tokens_kernel(const I* __restrict__ tok, int n, long V, int width,
                                                                      int* __restrict__ start, int* __restrict__ order, int* __restrict__ sorted) {
    extern __shared__ int hist[];                         // [SORT_WAVES][width], then this workgroup's scan
    __shared__ int below_s[SORT_WAVES], scan_s[SORT_WAVES];
    __shared__ int carry;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lo = (int)blockIdx.x * width, own = (int)(V - lo < width ? V - lo : width);
    for (int i = tid; i < SORT_WAVES * width; i += 64 * SORT_WAVES) hist[i] = 0;
    __syncthreads();
    const int piece = ((n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
    const int p0 = wave * piece, p1 = p0 + piece < n ? p0 + piece : n;
    int below = 0;
    int* mine = hist + wave * width;
    // the list 64 x BATCH tokens at a time, all loads of a batch on their way before the first is looked at: one after
    // the other they are a chain of L2 round trips (16,384 tokens: SORT_FIGURES)
    int ids[BATCH];
    const auto load = [&](int p) {
        I t[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) t[i] = p + 64 * i + lane < p1 ? tok[p + 64 * i + lane] : (I)-1;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) ids[i] = small_id(t[i]);
    };
    for (int p = p0; p < p1; p += 64 * BATCH) {
        load(p);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            below += (unsigned)ids[i] < (unsigned)lo ? 1 : 0;
            if ((unsigned)(ids[i] - lo) < (unsigned)own) atomicAdd(&mine[ids[i] - lo], 1);
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) below += __shfl_xor(below, off, 64);
    if (lane == 0) below_s[wave] = below;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) base += below_s[w];
    // exclusive scan of the ids' totals, 1024 at a time; each (wave, id) counter becomes its first place
    if (tid == 0) carry = base;
    for (int i0 = 0; i0 < own; i0 += 64 * SORT_WAVES) {
        const int i = i0 + tid;
        int total = 0;
        if (i < own)
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) total += hist[w * width + i];
        int inc = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(inc, off, 64);
            if (lane >= off) inc += t;
        }
        __syncthreads();                                  // scan_s and carry of the round before are read
        if (lane == 63) scan_s[wave] = inc;
        __syncthreads();
        int before = carry;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) before += w < wave ? scan_s[w] : 0;
        int at = before + inc - total;
        if (i < own) {
            start[lo + i] = at;
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                const int c = hist[w * width + i];
                hist[w * width + i] = at;
                at += c;
            }
            if (lo + i == V - 1) start[V] = at;
        }
        __syncthreads();
        if (tid == 64 * SORT_WAVES - 1) carry = before + inc;
    }
    __syncthreads();
    for (int p = p0; p < p1; p += 64 * BATCH) {
        if (piece > 64 * BATCH) load(p);                  // (else it is still there)
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int v = ids[i] - lo, q = p + 64 * i + lane;
            const bool hit = (unsigned)v < (unsigned)own;
            unsigned long long left = __ballot(hit);
            while (left != 0) {                           // one distinct id per turn
                const int lead = __ffsll((long long)left) - 1;
                const int u = __builtin_amdgcn_readlane(v, lead);
                const unsigned long long same = __ballot(hit && v == u) & left;
                const int at = mine[u];
                if (hit && v == u) {
                    const int to = at + __popcll(same & ((1ull << lane) - 1));
                    order[to] = q;
                    sorted[to] = ids[i];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (lane == lead) mine[u] = at + __popcll(same);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                left &= ~same;
            }
        }
    }
}

// partial[c][C] = sum of the 64 rows of chunk c of the sorted list, where they all belong to one id
__global__ __launch_bounds__(256) void sum_chunks_kernel(const int* __restrict__ order, const int* __restrict__ sorted, const int* __restrict__ start,
                                                         long V, const unsigned short* __restrict__ dy, float* __restrict__ partial, int C) {
    __shared__ float red[4][64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = blockIdx.x * CHUNK;
    if (s + CHUNK > start[V] || sorted[s] != sorted[s + CHUNK - 1]) return;
    const int nch = C / 8;
    for (int c0 = 0; c0 < nch; c0 += 64) {
        const int ch = c0 + lane;
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (ch < nch) {
#pragma unroll 8
            for (int i = 0; i < CHUNK / 4; ++i) {
                float f[8];
                const uint4 u = *(const uint4*)(dy + (long)order[s + wave * (CHUNK / 4) + i] * C + ch * 8);
                unpack8(u, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] += f[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) red[wave][lane * 8 + j] = acc[j];
        __syncthreads();
        for (int i = threadIdx.x; i < 512; i += 256)
            if (c0 * 8 + i < C) partial[(long)blockIdx.x * C + c0 * 8 + i] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
        __syncthreads();
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

// A thread has four channels in each half of the row: as many loads in flight as with eight together, and stores that leave no
// gaps between lanes.  The rows are stored past the caches, which they would only fill (ROWS_FIGURES).
// ADD: rows that some token names are added to dw (which another stream may be adding to as well: one atomic per element);
// otherwise every row is written
template <bool ADD>
__global__ __launch_bounds__(256) void sum_rows_kernel(const int* __restrict__ order, const int* __restrict__ start, const unsigned short* __restrict__ dy,
                                                       const float* __restrict__ partial, float* __restrict__ dw, long V, int C, float scale, int rows) {
    // a workgroup takes `rows` rows: only the place within them is divided, in 32 bits
    const int nch = C / 8;
    const long v0 = (long)blockIdx.x * rows;
    for (int i = threadIdx.x; i < rows * nch; i += 256) {
        const int dv = i / nch, c = (i - dv * nch) * 4;
        const long v = v0 + dv;
        if (v >= V) break;
        const int s = start[v], e = start[v + 1];
        floatx4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        const int c0 = (s + CHUNK - 1) / CHUNK, c1 = e / CHUNK;      // whole chunks of the segment
        if (partial == nullptr || c0 >= c1) {
            add_rows(acc, order, s, e, dy, C, c);
        } else {
            add_rows(acc, order, s, c0 * CHUNK, dy, C, c);
#pragma unroll 4
            for (int k = c0; k < c1; ++k) {
                acc[0] += *(const floatx4*)(partial + (long)k * C + c);
                acc[1] += *(const floatx4*)(partial + (long)k * C + c + C / 2);
            }
            add_rows(acc, order, c1 * CHUNK, e, dy, C, c);
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

// ids per workgroup of the sort: 256 workgroups where that leaves each at most 512 (32 KiB of counters)
inline int sort_width(long V) {
    const long w = (V + 255) / 256;
    return (int)(w > 512 ? 512 : w);
}

template <typename I>
void backward_of(const I* tok, const void* dy, float* dw, int add, long n, int C, long V, float scale, int* start, int* order, int* sorted,
                 float* partial, hipStream_t st) {
    const int width = sort_width(V);
    hipLaunchKernelGGL((sort_tokens_kernel<I>), dim3((unsigned)((V + width - 1) / width)), dim3(64 * SORT_WAVES), SORT_WAVES * width * sizeof(int), st,
                       tok, (int)n, V, width, start, order, sorted);
    if (partial != nullptr)
        hipLaunchKernelGGL(sum_chunks_kernel, dim3((unsigned)(n / CHUNK)), dim3(256), 0, st, order, sorted, start, V, (const unsigned short*)dy, partial, C);
    const int rows = C / 8 >= 512 ? 1 : 512 / (C / 8);
    const dim3 blocks((unsigned)((V + rows - 1) / rows));
    if (add)
        hipLaunchKernelGGL((sum_rows_kernel<true>), blocks, dim3(256), 0, st, order, start, (const unsigned short*)dy, partial, dw, V, C, scale, rows);
    else
        hipLaunchKernelGGL((sum_rows_kernel<false>), blocks, dim3(256), 0, st, order, start, (const unsigned short*)dy, partial, dw, V, C, scale, rows);
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

long token_embedding_chunks(long n) { return n >= 8 * CHUNK ? n / CHUNK : 0; }

void token_embedding_bwd(const void* tok, int tok64, const void* dy, float* dw, int add, long n, int C, long V, float scale, int* start, int* order,
                         int* sorted, float* partial, hipStream_t st) {
    if (tok64) backward_of((const int64_t*)tok, dy, dw, add, n, C, V, scale, start, order, sorted, partial, st);
    else backward_of((const int*)tok, dy, dw, add, n, C, V, scale, start, order, sorted, partial, st);
}

}  // namespace dpa
