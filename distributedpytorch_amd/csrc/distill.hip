// Distillation from a teacher's top logits, loss and gradient (gfx950).
//
//   q = softmax(z / tau) over the V classes of a row, p = softmax(t / tau) over the row's live teacher entries
//   (id in [0, V), t > -inf; an id may come twice);  row loss = tau^2 sum_k p_k (log p_k - log q_{id_k}), a row without
//   live entries gives 0;  loss = sum of the rows / N;   d loss / d z_j = tau / N (q_j - sum over k with id_k = j of p_k).
//
// Bound by memory: z is read once and its gradient written once, both by the forward call when a gradient will be asked
// for.  A 1024-thread workgroup takes a row.  Rows of up to 65,536 bf16 (32,768 fp32) columns stay in registers between the
// sweeps (maximum, sum, gradient); longer or unaligned ones are read again, from the caches where they fit.  The teacher's
// p is formed by the first wave from LDS; its share of the gradient - at most K places of a row - is written over the
// dense part behind a barrier, every place by all the entries that name it with the same sum, so that duplicates need
// neither an order nor an atomic.  Row losses are folded in a fixed order by a second small kernel.
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

constexpr int NT = 1024, KMAX = 1024;
constexpr float NEG_BIG = -1.0e30f, LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]);
template <> __device__ __forceinline__ void load8<unsigned short>(const unsigned short* p, float (&f)[8]) { const uint4 u = *(const uint4*)p; unpack8(u, f); }
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ float get1(const unsigned short* p) { return bf16_to_float(*p); }
__device__ __forceinline__ float get1(const float* p) { return *p; }
__device__ __forceinline__ void put1(unsigned short* p, float v) { *p = float_to_bf16(v); }
__device__ __forceinline__ void put1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store8(unsigned short* p, const float (&f)[8]) { *(uint4*)p = pack8(f); }
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
    *(float4*)(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_reduce_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, red[w]);
    return m;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_reduce_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += red[w];
    return s;
}

// live teacher entries of the row into LDS: ids_s (-1 where dead), p_s, logp_s.  Returns whether there are any.
__device__ __forceinline__ bool teacher_row(const DistillArgs& a, long row, int* ids_s, float* p_s, float* lp_s, float* red) {
    const int tid = threadIdx.x;
    float t = 0.f;
    bool live = false;
    if (tid < a.K) {
        const long id = a.ids64 ? (long)((const int64_t*)a.ids)[row * a.K + tid] : (long)((const int*)a.ids)[row * a.K + tid];
        t = a.teacher[row * a.K + tid];
        live = id >= 0 && id < a.V && !(t == -INFINITY);
        ids_s[tid] = live ? (int)id : -1;
    }
    const float m = block_max(live ? t : -INFINITY, red);
    const float x = live ? (t - m) * a.inv_tau : 0.f, e = live ? expf(x) : 0.f;
    const float s = block_sum(e, red);
    const bool any = __syncthreads_or(live);
    if (tid < a.K) {
        p_s[tid] = any ? e / s : 0.f;
        lp_s[tid] = any && live ? x - logf(s) : 0.f;
    }
    __syncthreads();
    return any;
}

// the row's loss (thread 0 writes it) and the teacher's places of the gradient; lse2 = log2 sum_j 2^(z_j c)
template <typename T>
__device__ __forceinline__ void finish_row(const DistillArgs& a, long row, const T* z, T* d, bool any, float c, float lse2, const int* ids_s, const float* p_s,
                                           const float* lp_s, float* red) {
    const int tid = threadIdx.x;
    float term = 0.f;
    if (any && tid < a.K && ids_s[tid] >= 0) {
        const int id = ids_s[tid];
        const float y = fmaf(get1(z + id), c, -lse2);                          // log2 q
        term = p_s[tid] == 0.f ? 0.f : p_s[tid] * (lp_s[tid] - y * LN2);
        if (d != nullptr) {
            float same = 0.f;
            for (int k = 0; k < a.K; ++k) same += ids_s[k] == id ? p_s[k] : 0.f;
            put1(d + id, (exp2f(y) - same) * a.grad_scale);
        }
    }
    const float sum = block_sum(term, red);
    if (tid == 0) a.row_loss[row] = any ? sum : 0.f;
}

// NCH > 0: the row in registers, NCH chunks of 8 per thread; 0: any length and alignment, read again for each sweep
template <typename T, int NCH>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
    __shared__ float red[NT / 64];
    __shared__ int ids_s[KMAX];
    __shared__ float p_s[KMAX], lp_s[KMAX];
    const int tid = threadIdx.x, V = a.V;
    const long row = blockIdx.x, ld = a.ld;
    const T* z = (const T*)a.logits + row * ld;
    T* d = a.dlogits != nullptr ? (T*)a.dlogits + row * ld : nullptr;
    const float c = a.inv_tau * LOG2E;
    if constexpr (NCH > 0) {
        constexpr int W = sizeof(T) == 2 ? 1 : 2;                              // 16-byte words of a chunk
        u32x4 raw[NCH][W];
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int i = (tid + k * NT) * 8;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                raw[k][w] = u32x4{0, 0, 0, 0};
                if (i < V) raw[k][w] = *(const u32x4*)((const unsigned char*)(z + i) + 16 * w);
            }
        }
        const bool any = teacher_row(a, row, ids_s, p_s, lp_s, red);           // while the row is on its way
        auto unpack = [&](int k, float (&f)[8]) {
            const int i = (tid + k * NT) * 8;
            if constexpr (sizeof(T) == 2) {
                unpack8(__builtin_bit_cast(uint4, raw[k][0]), f);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned u = raw[k][j >> 2][j & 3];                  // a scalar first: a bit cast of the element itself reads element 0
                    f[j] = __builtin_bit_cast(float, u);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = i + j < V ? f[j] : -INFINITY;
        };
        float m = NEG_BIG;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            float f[8];
            unpack(k, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, f[j]);
        }
        m = block_max(m, red) * c;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            float f[8];
            unpack(k, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += exp2f(fmaf(f[j], c, -m));
        }
        const float lse2 = m + log2f(block_sum(s, red));
        if (d != nullptr) {
            const float g = any ? a.grad_scale : 0.f;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                const int i = (tid + k * NT) * 8;
                if (i < ld) {
                    float f[8];
                    unpack(k, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = any && i + j < V ? exp2f(fmaf(f[j], c, -lse2)) * g : 0.f;
                    store8(d + i, f);
                }
            }
            __syncthreads();                                                   // the dense part is there before the teacher's places
        }
        finish_row<T>(a, row, z, d, any, c, lse2, ids_s, p_s, lp_s, red);
    } else {
        const bool any = teacher_row(a, row, ids_s, p_s, lp_s, red);
        const int nv = a.aligned ? V / 8 : 0;
        float m = NEG_BIG, s = 0.f;
        for (int i = tid; i < nv; i += NT) {
            float f[8];
            load8(z + i * 8, f);
            float lm = m;
#pragma unroll
            for (int j = 0; j < 8; ++j) lm = fmaxf(lm, f[j] * c);
            s *= exp2f(m - lm);
            m = lm;
#pragma unroll
            for (int j = 0; j < 8; ++j) s += exp2f(fmaf(f[j], c, -m));
        }
        for (int i = nv * 8 + tid; i < V; i += NT) {
            const float x = get1(z + i), lm = fmaxf(m, x * c);
            s = s * exp2f(m - lm) + exp2f(fmaf(x, c, -lm));
            m = lm;
        }
        const float mb = block_max(m, red);
        const float lse2 = mb + log2f(block_sum(s * exp2f(m - mb), red));
        if (d != nullptr) {
            const float g = any ? a.grad_scale : 0.f;
            for (int i = tid; i < nv; i += NT) {
                float f[8];
                load8(z + i * 8, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = any ? exp2f(fmaf(f[j], c, -lse2)) * g : 0.f;
                store8(d + i * 8, f);
            }
            for (long i = nv * 8 + tid; i < ld; i += NT) put1(d + i, any && i < V ? exp2f(fmaf(get1(z + i), c, -lse2)) * g : 0.f);
            __syncthreads();
        }
        finish_row<T>(a, row, z, d, any, c, lse2, ids_s, p_s, lp_s, red);
    }
}

// loss = scale * sum of the rows, one workgroup, fixed order
__global__ __launch_bounds__(NT) void fold_rows_kernel(const float* __restrict__ row_loss, long n, float scale, float* __restrict__ loss) {
    __shared__ float red[NT / 64];
    float s = 0.f;
    for (long i = threadIdx.x; i < n; i += NT) s += row_loss[i];
    s = block_sum(s, red);
    if (threadIdx.x == 0) *loss = s * scale;
}

// d *= *g unless *g is 1
template <typename T>
__global__ __launch_bounds__(256) void scale_grad_kernel(T* __restrict__ d, const float* __restrict__ g, long n) {
    const float gs = *g;
    if (gs == 1.f) return;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) put1(d + i, get1(d + i) * gs);
}

template <typename T>
void launch(const DistillArgs& a, hipStream_t st) {
    const int nch = (int)((a.ld + 8 * NT - 1) / (8 * NT));
    const bool held = a.aligned && a.ld % 8 == 0 && nch <= (sizeof(T) == 2 ? 8 : 4);
#define DPA_DISTILL(N_) hipLaunchKernelGGL((distill_kernel<T, N_>), dim3((unsigned)a.N), dim3(NT), 0, st, a)
    if (!held) { DPA_DISTILL(0); return; }
    if constexpr (sizeof(T) == 2) {
        switch (nch) {
            case 1: DPA_DISTILL(1); break;
            case 2: DPA_DISTILL(2); break;
            case 3: DPA_DISTILL(3); break;
            case 4: DPA_DISTILL(4); break;
            case 5: DPA_DISTILL(5); break;
            case 6: DPA_DISTILL(6); break;
            case 7: DPA_DISTILL(7); break;
            default: DPA_DISTILL(8); break;
        }
    } else {
        switch (nch) {
            case 1: DPA_DISTILL(1); break;
            case 2: DPA_DISTILL(2); break;
            case 3: DPA_DISTILL(3); break;
            default: DPA_DISTILL(4); break;
        }
    }
#undef DPA_DISTILL
}

}  // namespace

int distill_max_entries() { return KMAX; }

void distill(const DistillArgs& a, int is_bf16, float loss_scale, float* loss, hipStream_t st) {
    if (a.N > 0) {
        if (is_bf16) launch<unsigned short>(a, st);
        else launch<float>(a, st);
    }
    hipLaunchKernelGGL(fold_rows_kernel, dim3(1), dim3(NT), 0, st, a.row_loss, a.N, loss_scale, loss);
}

void scale_grad(void* d, int is_bf16, const float* g, long n, hipStream_t st) {
    long b = (n + 255) / 256;
    const unsigned blocks = (unsigned)(b < 1 ? 1 : b > 4096 ? 4096 : b);
    if (is_bf16) hipLaunchKernelGGL((scale_grad_kernel<unsigned short>), dim3(blocks), dim3(256), 0, st, (unsigned short*)d, g, n);
    else hipLaunchKernelGGL((scale_grad_kernel<float>), dim3(blocks), dim3(256), 0, st, (float*)d, g, n);
}

}  // namespace dpa
