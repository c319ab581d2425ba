// Distillation from a teacher's top logits, loss and gradient (gfx950).
//
//   q = softmax(z / tau) over the V classes of a row, p = softmax(t / tau) over the row's live teacher entries
//   (id in [0, V), t > -inf; an id may come twice);  row loss = tau^2 sum_k p_k (log p_k - log q_{id_k}), a row without
//   live entries gives 0;  loss = sum of the rows / N;   d loss / d z_j = tau / N (q_j - sum over k with id_k = j of p_k).
//
// Bound by memory: z is read once and its gradient written once, both by the forward call when a gradient will be asked
// for.  A workgroup takes a row, held between the sweeps (maximum, sum of exponentials, gradient) as the 16-byte vectors
// it was read in - rows of any length and start are covered by the aligned vectors over them, the two at the ends element
// by element.  Four builds, chosen by how many vectors a row has (`launch`):
//   up to 1024     256 threads, registers: short rows are all latency, and fewer waves meet at fewer, cheaper barriers;
//   up to 8192     1024 threads, registers, as many workgroups as the CUs hold and the next row's loads in flight under this
//                  row's arithmetic: one workgroup fills a CU here, and a row's load, sweeps and store would follow one
//                  another (16,384 rows of 50,257 bf16: 1083 us so, 819 in flight; a large copy of the same bytes takes 690);
//   up to 25,600   1024 threads, 17 vectors a thread in registers and up to 8 in LDS (2047 rows of 100,001 fp32: 425 us,
//                  read again for the gradient 711);
//   beyond         read again for the gradient.
// The teacher's p goes through LDS; its share of the gradient - at most K places of a row - is written over the dense part
// behind a barrier, every place by all the entries that name it with the same sum, so that duplicates need neither an
// order nor an atomic.  The loss is folded in a fixed order by a second small kernel.
// The forward writes the gradient for an upstream gradient of 1.  Backward starts the same kernel with the real one: where that is 1
// nothing is done, and otherwise the gradient is formed again from the logits, which crosses memory as often as scaling the
// written one would and rounds once.
#include <stdexcept>
#include <string>
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

constexpr int KMAX = 1024;
constexpr float LOWEST = -3.4028234664e38f, LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float get1(const unsigned short* p) { return bf16_to_float(*p); }
__device__ __forceinline__ float get1(const float* p) { return *p; }
__device__ __forceinline__ void put1(unsigned short* p, float v) { *p = float_to_bf16(v); }
__device__ __forceinline__ void put1(float* p, float v) { *p = v; }
// 2^x as one instruction; arguments are <= 0 up to rounding, and what lies below the normal numbers may be 0
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T> struct Vec;
template <> struct Vec<unsigned short> {
    static constexpr int N = 8;
    static constexpr unsigned NONE = 0xff80ff80u;                              // -inf, twice
    __device__ static void unpack(const u32x4& r, float (&f)[8]) { unpack8(__builtin_bit_cast(uint4, r), f); }
    __device__ static u32x4 pack(const float (&f)[8]) { return __builtin_bit_cast(u32x4, pack8(f)); }
    __device__ static void set(u32x4& r, int j, unsigned short v) { r[j >> 1] = (j & 1) ? ((r[j >> 1] & 0xffffu) | ((unsigned)v << 16)) : ((r[j >> 1] & 0xffff0000u) | v); }
};
template <> struct Vec<float> {
    static constexpr int N = 4;
    static constexpr unsigned NONE = 0xff800000u;
    __device__ static void unpack(const u32x4& r, float (&f)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned u = r[j];                                           // a scalar first: a bit cast of the element itself reads element 0
            f[j] = __builtin_bit_cast(float, u);
        }
    }
    __device__ static u32x4 pack(const float (&f)[4]) {
        return u32x4{__builtin_bit_cast(unsigned, f[0]), __builtin_bit_cast(unsigned, f[1]), __builtin_bit_cast(unsigned, f[2]), __builtin_bit_cast(unsigned, f[3])};
    }
    __device__ static void set(u32x4& r, int j, float v) { r[j] = __builtin_bit_cast(unsigned, v); }
};

// One row as the aligned 16-byte vectors over it: vector i holds elements N i - lead ..
template <typename T>
struct Row {
    const T* z;
    T* d;
    int lead, V, ld;
    __device__ __forceinline__ Row(const DistillArgs& a, long row) : z((const T*)a.logits + row * a.ld),
        d(a.dlogits != nullptr ? (T*)a.dlogits + row * a.ld : nullptr), lead((int)(((uintptr_t)z & 15) / sizeof(T))), V(a.V), ld((int)a.ld) {}
    // columns past the classes as -inf: they take part in nothing.  WHOLE: rows are whole vectors, and where the caller is
    // `sure` that vector i lies in the row the access stands in no branch - behind one the compiler no longer knows how many
    // stores follow a load and waits for them all in front of the next row.
    template <bool WHOLE>
    __device__ __forceinline__ u32x4 load(int i, bool sure) const {
        if (WHOLE) {
            u32x4 r = {Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE};
            const int e = i * Vec<T>::N;
            if (sure || e < ld) r = *(const u32x4*)(z + e);
            if (e + Vec<T>::N > V) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    constexpr int P = Vec<T>::N / 4;                           // values of a word
                    const unsigned u = r[w], none = Vec<T>::NONE;
                    if (P == 1) r[w] = e + w < V ? u : none;
                    else r[w] = (e + 2 * w < V ? u & 0xffffu : none & 0xffffu) | (e + 2 * w + 1 < V ? u & 0xffff0000u : none & 0xffff0000u);
                }
            }
            return r;
        }
        const int e = i * Vec<T>::N - lead;
        if (e >= 0 && e + Vec<T>::N <= V) return *(const u32x4*)(z + e);
        u32x4 r = {Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE};
        if (e < V && e > -Vec<T>::N)
#pragma unroll
            for (int j = 0; j < Vec<T>::N; ++j)
                if (e + j >= 0 && e + j < V) Vec<T>::set(r, j, z[e + j]);
        return r;
    }
    template <bool WHOLE>
    __device__ __forceinline__ void store(int i, const float (&f)[Vec<T>::N], bool sure) const {
        if (WHOLE) {
            if (sure || i * Vec<T>::N < ld) *(u32x4*)(d + i * Vec<T>::N) = Vec<T>::pack(f);
            return;
        }
        const int e = i * Vec<T>::N - lead;
        if (e >= 0 && e + Vec<T>::N <= ld) { *(u32x4*)(d + e) = Vec<T>::pack(f); return; }
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j)
            if (e + j >= 0 && e + j < ld) put1(d + e + j, f[j]);
    }
};

// Two reductions over the workgroup in one exchange; every call in a row of `red` of its own, so one barrier each
template <int NW, bool MAX>
__device__ __forceinline__ float2 fold2(float x, float y, float2* red) {
    x = MAX ? wave_reduce_max(x) : wave_reduce_sum(x);
    y = MAX ? wave_reduce_max(y) : wave_reduce_sum(y);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(x, y);
    __syncthreads();
    float2 s = red[threadIdx.x % NW];
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) {
        const float vx = __shfl_xor(s.x, off, 64), vy = __shfl_xor(s.y, off, 64);
        s.x = MAX ? fmaxf(s.x, vx) : s.x + vx;
        s.y = MAX ? fmaxf(s.y, vy) : s.y + vy;
    }
    return s;
}

// KE = teacher entries per thread
template <int KE> struct Teacher { int id[KE]; float t[KE], z[KE]; };
template <int NT, int KE>
__device__ __forceinline__ void load_teacher(const DistillArgs& a, long row, Teacher<KE>& e) {
#pragma unroll
    for (int i = 0; i < KE; ++i) {
        const int k = threadIdx.x + i * NT;
        e.id[i] = -1;
        e.t[i] = 0.f;
        if (k < a.K) {
            const long id = a.ids64 ? (long)((const int64_t*)a.ids)[row * a.K + k] : (long)((const int*)a.ids)[row * a.K + k];
            e.t[i] = a.teacher[row * a.K + k];
            e.id[i] = id >= 0 && id < a.V ? (int)id : -1;
        }
    }
}
template <typename T, int KE>
__device__ __forceinline__ void load_student(const T* z, Teacher<KE>& e) {
#pragma unroll
    for (int i = 0; i < KE; ++i) {
        if (e.t[i] == -INFINITY) e.id[i] = -1;
        e.z[i] = e.id[i] >= 0 ? get1(z + e.id[i]) : 0.f;
    }
}

// NREG vectors a thread in registers; LDS: more of them in LDS; PIPE: the next row's loads go out before this row's sweeps;
// NREG = 0: nothing is kept.  A row has more than NT (NREG - 1) vectors, with LDS more than 8 NT.
template <typename T, int NT, int NREG, bool LDS, bool PIPE, bool WHOLE>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
    constexpr int N = Vec<T>::N, NW = NT / 64, KE = (KMAX + NT - 1) / NT, HELD = NREG > 0 ? NREG : 1, SURE = LDS ? 8 : HELD - 1;
    extern __shared__ __attribute__((aligned(16))) u32x4 more[];               // LDS: vectors NREG .. of every thread
    __shared__ float2 red[3][NW];
    __shared__ int ids_s[KMAX];
    __shared__ float p_s[KMAX];
    const int tid = threadIdx.x;
    const float c = a.inv_tau * LOG2E, up = a.upstream != nullptr ? *a.upstream : 1.f, grad_scale = a.grad_scale * up;
    if (a.unless_one && up == 1.f) return;                                     // the whole launch: the gradient is there already
    u32x4 raw[HELD], nraw[PIPE ? HELD : 1];
    Teacher<KE> te, nte;
    float total = 0.f;
    long row = blockIdx.x;
    if (row < a.N) {
        const Row<T> r(a, row);
        load_teacher<NT>(a, row, te);
        if (NREG > 0 && PIPE)
#pragma unroll
            for (int k = 0; k < HELD; ++k) raw[k] = r.template load<WHOLE>(tid + k * NT, k < SURE);
        load_student(r.z, te);
    }
    for (; row < a.N; row += gridDim.x) {
        const Row<T> r(a, row);
        const int nv = (r.lead + r.ld + N - 1) / N;
        const long next = row + gridDim.x;
        if (NREG > 0 && !PIPE)
#pragma unroll
            for (int k = 0; k < HELD; ++k) raw[k] = r.template load<WHOLE>(tid + k * NT, k < SURE);
        if (LDS)
            for (int k = NREG; tid + k * NT < nv; ++k) more[(k - NREG) * NT + tid] = r.template load<WHOLE>(tid + k * NT, true);
        if (next < a.N) {
            load_teacher<NT>(a, next, nte);
            if (NREG > 0 && PIPE) {
                const Row<T> rn(a, next);
#pragma unroll
                for (int k = 0; k < HELD; ++k) nraw[k] = rn.template load<WHOLE>(tid + k * NT, k < SURE);
            }
        }
        const auto sweep = [&](auto&& f) {                                     // f(vector number, its values, whether the row surely has it)
            if (NREG > 0) {
#pragma unroll
                for (int k = 0; k < HELD; ++k) {
                    u32x4 q = raw[k];
                    asm volatile("" : "+v"(q));                                // unpacked anew in every sweep, not kept as floats between them
                    float v[N];
                    Vec<T>::unpack(q, v);
                    f(tid + k * NT, v, k < SURE);
                }
                if (LDS)
                    for (int k = NREG; tid + k * NT < nv; ++k) {
                        float v[N];
                        Vec<T>::unpack(more[(k - NREG) * NT + tid], v);
                        f(tid + k * NT, v, true);
                    }
            } else {
                for (int i = tid; i < nv; i += NT) {
                    float v[N];
                    Vec<T>::unpack(r.template load<WHOLE>(i, true), v);
                    f(i, v, true);
                }
            }
        };
        // maxima of the row and of the teacher's live entries (a NaN entry is live: the row's sums become NaN)
        float m = LOWEST, s = 0.f, tm = -INFINITY;
        bool live = false;
#pragma unroll
        for (int i = 0; i < KE; ++i)
            if (te.id[i] >= 0) { live = true; tm = fmaxf(tm, te.t[i]); }
        if (NREG > 0) {
            sweep([&](int, float (&v)[N], bool) {
#pragma unroll
                for (int j = 0; j < N; ++j) m = fmaxf(m, v[j]);
            });
        } else {                                                               // maximum and sum in one reading
            sweep([&](int, float (&v)[N], bool) {
                float lm = m;
#pragma unroll
                for (int j = 0; j < N; ++j) lm = fmaxf(lm, v[j]);
                s *= fast_exp2((m - lm) * c);
                m = lm;
#pragma unroll
                for (int j = 0; j < N; ++j) s += fast_exp2((v[j] - m) * c);
            });
        }
        const float2 mm = fold2<NW, true>(m, tm, red[0]);
        // Exponents are differences from the maximum, and the sum divides: with the sum's logarithm added to the maximum instead, q
        // would be half a place of the maximum off (fp32 logits around 1000: 4e-5 of q, 1e-7 so).  Where one multiply-add forms them,
        // what m2's rounding takes moves all of a row's exponents alike and leaves with the sum - as long as it is small: rows that are far
        // from zero (masked as a whole with the type's lowest value, say) have the difference formed first, and so has a row that is
        // read again, whose sum is made by parts from other maxima.  (For every row: 851 instead of 808 us at 16,384 x 50,257.)
        const float mx = mm.x, m2 = mx * c;
        const bool far = NREG == 0 || !(fabsf(m2) < 1e6f);                     // the same for the whole workgroup
        const auto near_exponent = [&](float v) { return fmaf(v, c, -m2); };
        const auto far_exponent = [&](float v) { return (v - mx) * c; };
        const auto exponent = [&](float v) { return far ? far_exponent(v) : near_exponent(v); };
        const auto with_exponent = [&](auto&& body) {                          // not chosen element by element
            if (far) body(far_exponent);
            else body(near_exponent);
        };
        if (NREG > 0)
            with_exponent([&](auto&& e) {
                sweep([&](int, float (&v)[N], bool) {
#pragma unroll
                    for (int j = 0; j < N; ++j) s += fast_exp2(e(v[j]));
                });
            });
        else
            s *= fast_exp2((m - mx) * c);
        float x[KE], ts = 0.f;
#pragma unroll
        for (int i = 0; i < KE; ++i) {
            x[i] = te.id[i] >= 0 ? (te.t[i] - mm.y) * a.inv_tau : 0.f;
            ts += te.id[i] >= 0 ? expf(x[i]) : 0.f;
        }
        const float2 ss = fold2<NW, false>(s, ts, red[1]);
        const bool any = __syncthreads_or(live);                               // a row without a teacher gives nothing, whatever it holds
        const float inv = 1.f / ss.x, lsum = log2f(ss.x);
        float p[KE], term = 0.f;
#pragma unroll
        for (int i = 0; i < KE; ++i) {
            const int k = tid + i * NT;
            p[i] = te.id[i] >= 0 ? expf(x[i]) / ss.y : 0.f;
            if (k < a.K) { ids_s[k] = te.id[i]; p_s[k] = p[i]; }
            const float y = exponent(te.z[i]) - lsum;                          // log2 q
            if (te.id[i] >= 0) term += p[i] == 0.f ? 0.f : p[i] * (x[i] - logf(ss.y) - y * LN2);
        }
        if (next < a.N) load_student((const T*)a.logits + next * a.ld, nte);
        if (r.d != nullptr) {
            const float g = grad_scale * inv;
            if (any)
                with_exponent([&](auto&& e) {
                    sweep([&](int i, float (&v)[N], bool sure) {
#pragma unroll
                        for (int j = 0; j < N; ++j) v[j] = fast_exp2(e(v[j])) * g;
                        r.template store<WHOLE>(i, v, sure);
                    });
                });
            else
                for (int i = tid; i < nv; i += NT) {
                    float v[N] = {};
                    r.template store<WHOLE>(i, v, true);
                }
        }
        term = fold2<NW, false>(term, 0.f, red[2]).x;                          // (and: the dense part and the teacher's p are there)
        if (r.d != nullptr)
#pragma unroll
            for (int i = 0; i < KE; ++i)
                if (te.id[i] >= 0) {
                    float same = 0.f;
                    for (int k = 0; k < a.K; ++k) same += ids_s[k] == te.id[i] ? p_s[k] : 0.f;
                    put1(r.d + te.id[i], (fast_exp2(exponent(te.z[i])) * inv - same) * grad_scale);
                }
        if (any) total += term;
        __syncthreads();                                                       // ids_s and p_s are read
        te = nte;
        if (NREG > 0 && PIPE)
#pragma unroll
            for (int k = 0; k < HELD; ++k) raw[k] = nraw[k];
    }
    if (tid == 0 && a.row_loss != nullptr) a.row_loss[blockIdx.x] = total;
}

// loss = scale * sum of the workgroups' shares, fixed order
__global__ __launch_bounds__(256) void fold_loss_kernel(const float* __restrict__ part, int n, float scale, float* __restrict__ loss) {
    __shared__ float2 red[4];
    float s = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    s = fold2<4, false>(s, 0.f, red).x;
    if (threadIdx.x == 0) *loss = s * scale;
}

template <typename T, int NT, int NREG, bool LDS, bool PIPE, bool WHOLE>
void start_one(const DistillArgs& a, int blocks, int lds, hipStream_t st) {
    if (LDS) {                                                                 // for every call: the limit belongs to the current device
        const hipError_t e = hipFuncSetAttribute((const void*)distill_kernel<T, NT, NREG, LDS, PIPE, WHOLE>, hipFuncAttributeMaxDynamicSharedMemorySize, 8 * 1024 * 16);
        if (e != hipSuccess) throw std::runtime_error(std::string("distill: no LDS for a wide row: ") + hipGetErrorString(e));
    }
    hipLaunchKernelGGL((distill_kernel<T, NT, NREG, LDS, PIPE, WHOLE>), dim3((unsigned)blocks), dim3(NT), lds, st, a);
}
template <typename T, int NT, int NREG, bool LDS, bool PIPE>
void start(const DistillArgs& a, int blocks, int lds, hipStream_t st) {
    if (a.ld % Vec<T>::N == 0) start_one<T, NT, NREG, LDS, PIPE, true>(a, blocks, lds, st);
    else start_one<T, NT, NREG, LDS, PIPE, false>(a, blocks, lds, st);
}

// 16-byte vectors that cover any row, its start anywhere in one
template <typename T>
long vectors(long ld) { return (ld + Vec<T>::N - 1) / Vec<T>::N + (ld % Vec<T>::N != 0); }

template <typename T>
int blocks_of(long N, long ld) {
    const long v = vectors<T>(ld), cus = 256;
    const long most = v <= 1024 ? 4096 : v <= 8192 ? (v <= 3 * 1024 ? 2 * cus : cus) : 4 * cus;
    return (int)(N < most ? N : most);
}

template <typename T>
void launch(const DistillArgs& a, int blocks, hipStream_t st) {
    const long v = vectors<T>(a.ld);
    if (v <= 1024) {
        switch ((v + 255) / 256) {
            case 1: start<T, 256, 1, false, false>(a, blocks, 0, st); break;
            case 2: start<T, 256, 2, false, false>(a, blocks, 0, st); break;
            case 3: start<T, 256, 3, false, false>(a, blocks, 0, st); break;
            default: start<T, 256, 4, false, false>(a, blocks, 0, st); break;
        }
    } else if (v <= 8192) {
        switch ((v + 1023) / 1024) {
            case 2: start<T, 1024, 2, false, true>(a, blocks, 0, st); break;
            case 3: start<T, 1024, 3, false, true>(a, blocks, 0, st); break;
            case 4: start<T, 1024, 4, false, true>(a, blocks, 0, st); break;
            case 5: start<T, 1024, 5, false, true>(a, blocks, 0, st); break;
            case 6: start<T, 1024, 6, false, true>(a, blocks, 0, st); break;
            case 7: start<T, 1024, 7, false, true>(a, blocks, 0, st); break;
            default: start<T, 1024, 8, false, true>(a, blocks, 0, st); break;
        }
    } else if (v <= 25 * 1024) {
        const long over = v - 17 * 1024;
        start<T, 1024, 17, true, false>(a, blocks, over > 0 ? (int)((over + 1023) / 1024) * 1024 * 16 : 0, st);
    } else {
        start<T, 1024, 0, false, false>(a, blocks, 0, st);
    }
}

}  // namespace

int distill_max_entries() { return KMAX; }

int distill_blocks(int is_bf16, long N, long ld) { return is_bf16 ? blocks_of<unsigned short>(N, ld) : blocks_of<float>(N, ld); }

void distill(const DistillArgs& a, int is_bf16, float loss_scale, float* loss, hipStream_t st) {
    const int blocks = distill_blocks(is_bf16, a.N, a.ld);
    if (blocks > 0) {
        if (is_bf16) launch<unsigned short>(a, blocks, st);
        else launch<float>(a, blocks, st);
    }
    if (loss != nullptr) hipLaunchKernelGGL(fold_loss_kernel, dim3(1), dim3(256), 0, st, a.row_loss, blocks, loss_scale, loss);
}

}  // namespace dpa
