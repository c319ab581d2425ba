// Norm of every query and key head and the rotation by position in one pass over the packed projection, forward and
// backward (gfx950).
//
//   x: one head of one token, D channels;  r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = w n  (without weights: y = x),
//   pairs (a, b) of the first R channels:  (a', b') = (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i];
//   half-split pairs are channels (i, i + R/2), interleaved ones (2i, 2i + 1).
//   Backward: g = the gradient rotated by -t;  dx = r (g w - n mean(g w n)),  dw = sum over tokens and heads of g n.
//
// Both directions are bound by memory: q and k are read once and written once (values stay where the projection put them;
// only their gradient is copied into the packed one).  A wave takes one token and walks its heads, 16 bytes a lane, so a
// token's R/2 angles are made once - one per lane, in 64 bits (a position times a frequency in turns keeps the fraction that
// matters at any position, where 32 bits have lost it past some 10^4), then sine and cosine of the fraction in 32 - and
// handed round through LDS.  Reductions over a head are shuffles inside its 4 to 32 lanes.  The gains' gradients stay in
// registers over all of a wave's tokens and are folded per workgroup, then over workgroups in a fixed order: no atomics.
#include "common.h"
#include "kernels.h"

namespace dpa {
namespace {

constexpr int WAVES = 4, AHEAD = 6;
constexpr double INV_2PI = 0.15915494309189533577;

// orders one lane's LDS accesses with another's of the same wave
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// cos / sin of the token's angles into this wave's LDS row (R / 2 <= 128 of them)
__device__ __forceinline__ void make_angles(float2* cs, const double* __restrict__ inv_freq, int half, long pos, int lane) {
    for (int i = lane; i < half; i += 64) {
        double t = (double)pos * inv_freq[i] * INV_2PI;
        t -= rint(t);
        float s, c;
        sincospif(2.f * (float)t, &s, &c);
        cs[i] = make_float2(c, s);
    }
}

// rotates the 8 channels of this lane (channels 8 ch ..), partner values from the lane that holds the other half; `sign` -1 turns back
template <bool INTER>
__device__ __forceinline__ void rotate8(float (&v)[8], const float2* cs, int ch, int R, int lane_base, float sign) {
    const int hc = R / 16;                                // chunks of half the rotated channels
    if (INTER) {
        if (ch * 8 < R) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = cs[ch * 4 + i];
                const float a = v[2 * i], b = v[2 * i + 1], s = sign * t.y;
                v[2 * i] = a * t.x - b * s;
                v[2 * i + 1] = b * t.x + a * s;
            }
        }
    } else {
        const bool rot = ch < 2 * hc, low = ch < hc;
        const int pch = rot ? (low ? ch + hc : ch - hc) : ch;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __shfl(v[i], lane_base + pch, 64);
        if (rot) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 t = cs[(low ? ch : pch) * 8 + i];
                const float s = low ? -sign * t.y : sign * t.y;
                v[i] = v[i] * t.x + o[i] * s;
            }
        }
    }
}

template <int L>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// L lanes per head (D <= 8 L)
template <int L, bool NORM, bool INTER>
__global__ __launch_bounds__(64 * WAVES) void heads_fwd_kernel(HeadsArgs a, unsigned short* __restrict__ q, unsigned short* __restrict__ k) {
    __shared__ float2 cs_all[WAVES][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ch = lane % L, sub = lane / L, base = lane - ch;
    const bool in = ch * 8 < a.D;
    float wq[8], wk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        wq[i] = NORM && in ? a.qw[ch * 8 + i] : 1.f;
        wk[i] = NORM && in ? a.kw[ch * 8 + i] : 1.f;
    }
    float2* cs = cs_all[wave];
    const int nh = a.Hq + a.Hkv;
    const long row = (long)(a.Hq + 2 * a.Hkv) * a.D;
    for (long tok = (long)blockIdx.x * WAVES + wave; tok < a.tokens; tok += (long)gridDim.x * WAVES) {
        const unsigned short* x = (const unsigned short*)a.qkv + tok * row;
        for (int h0 = 0; h0 < nh; h0 += AHEAD * (64 / L)) {
            uint4 u[AHEAD];                                // on their way while the angles are made
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int hd = h0 + i * (64 / L) + sub;
                u[i] = make_uint4(0, 0, 0, 0);
                if (in && hd < nh) u[i] = *(const uint4*)(x + (long)hd * a.D + ch * 8);
            }
            if (h0 == 0 && a.R > 0) make_angles(cs, a.inv_freq, a.R / 2, a.positions != nullptr ? a.positions[tok] : tok % a.T, lane);
            wave_sync();
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int hd = h0 + i * (64 / L) + sub;
                if (h0 + i * (64 / L) >= nh) break;
                const bool live = in && hd < nh, is_q = hd < a.Hq;
                float v[8];
                unpack8(u[i], v);
                if (NORM) {
                    float s = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) s += v[j] * v[j];
                    const float r = rsqrtf(head_sum<L>(s) / (float)a.D + a.eps);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= r * (is_q ? wq[j] : wk[j]);
                }
                if (a.R > 0) rotate8<INTER>(v, cs, ch, a.R, base, 1.f);
                if (live) {
                    unsigned short* dst = is_q ? q + (tok * a.Hq + hd) * a.D : k + (tok * a.Hkv + hd - a.Hq) * a.D;
                    *(uint4*)(dst + ch * 8) = pack8(v);
                }
            }
        }
        wave_sync();
    }
}

// partial [2][gridDim.x][D]: this workgroup's share of dqw and dkw
template <int L, bool NORM, bool INTER>
__global__ __launch_bounds__(64 * WAVES) void heads_bwd_kernel(HeadsArgs a, const unsigned short* __restrict__ dq, const unsigned short* __restrict__ dk,
                                                               const unsigned short* __restrict__ dv, unsigned short* __restrict__ dqkv,
                                                               float* __restrict__ partial) {
    __shared__ float2 cs_all[WAVES][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ch = lane % L, sub = lane / L, base = lane - ch;
    const bool in = ch * 8 < a.D;
    float wq[8], wk[8], gq[8], gk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        wq[i] = NORM && in ? a.qw[ch * 8 + i] : 1.f;
        wk[i] = NORM && in ? a.kw[ch * 8 + i] : 1.f;
        gq[i] = gk[i] = 0.f;
    }
    float2* cs = cs_all[wave];
    const int nh = a.Hq + a.Hkv, all = nh + a.Hkv;
    const long row = (long)all * a.D;
    for (long tok = (long)blockIdx.x * WAVES + wave; tok < a.tokens; tok += (long)gridDim.x * WAVES) {
        if (a.R > 0) make_angles(cs, a.inv_freq, a.R / 2, a.positions != nullptr ? a.positions[tok] : tok % a.T, lane);
        wave_sync();
        const unsigned short* x = (const unsigned short*)a.qkv + tok * row;
        unsigned short* dx = dqkv + tok * row;
        for (int h0 = 0; h0 < all; h0 += 64 / L) {
            const int hd = h0 + sub;
            const bool live = in && hd < all, is_q = hd < a.Hq, is_v = hd >= nh;
            float g[8] = {0, 0, 0, 0, 0, 0, 0, 0}, n[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            uint4 u = make_uint4(0, 0, 0, 0);
            if (live) {
                const unsigned short* src = is_q ? dq + (tok * a.Hq + hd) * a.D
                                                 : is_v ? dv + (tok * a.Hkv + hd - nh) * a.D : dk + (tok * a.Hkv + hd - a.Hq) * a.D;
                u = *(const uint4*)(src + ch * 8);
                // a value's gradient is copied as it is and enters no sum: it may be infinite.  (Selected: a branch around the
                // unpacking has the loads behind it wait, 112 -> 120 us at 2 x 8191 x 24 heads of 128.)
                unpack8(make_uint4(is_v ? 0 : u.x, is_v ? 0 : u.y, is_v ? 0 : u.z, is_v ? 0 : u.w), g);
                if (NORM && !is_v) { const uint4 w = *(const uint4*)(x + (long)hd * a.D + ch * 8); unpack8(w, n); }
            }
            if (a.R > 0) rotate8<INTER>(g, cs, ch, a.R, base, -1.f);
            if (NORM) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += n[i] * n[i];
                // lanes without a query or key head add nothing to the gains' sums (with eps = 0 their 1 / sqrt is infinite)
                const float ms = head_sum<L>(s) / (float)a.D + a.eps, r = live && !is_v ? rsqrtf(ms) : 0.f;
                float d = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    n[i] *= r;
                    const float gn = g[i] * n[i];
                    if (is_q) gq[i] += gn; else gk[i] += gn;       // a value head has g = n = 0
                    g[i] *= is_q ? wq[i] : wk[i];
                    d += g[i] * n[i];
                }
                d = head_sum<L>(d) / (float)a.D;
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = r * (g[i] - n[i] * d);
            }
            if (live) *(uint4*)(dx + (long)hd * a.D + ch * 8) = is_v ? u : pack8(g);
        }
        wave_sync();
    }
    if (!NORM) return;
    // the 64 / L heads that share a channel, then the waves, then one partial row per workgroup
    __shared__ float red[2][WAVES][L * 8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int off = L; off < 64; off <<= 1) {
            gq[i] += __shfl_xor(gq[i], off, 64);
            gk[i] += __shfl_xor(gk[i], off, 64);
        }
        if (sub == 0) { red[0][wave][ch * 8 + i] = gq[i]; red[1][wave][ch * 8 + i] = gk[i]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += 64 * WAVES) {
        const int which = i / a.D, c = i - which * a.D;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += red[which][w][c];
        partial[((long)which * gridDim.x + blockIdx.x) * a.D + c] = s;
    }
}

template <int L>
void fwd_of(const HeadsArgs& a, unsigned short* q, unsigned short* k, unsigned blocks, hipStream_t st) {
#define DPA_HEADS(N_, I_) hipLaunchKernelGGL((heads_fwd_kernel<L, N_, I_>), dim3(blocks), dim3(64 * WAVES), 0, st, a, q, k)
    if (a.qw != nullptr) { if (a.interleaved) DPA_HEADS(true, true); else DPA_HEADS(true, false); }
    else { if (a.interleaved) DPA_HEADS(false, true); else DPA_HEADS(false, false); }
#undef DPA_HEADS
}
template <int L>
void bwd_of(const HeadsArgs& a, const unsigned short* dq, const unsigned short* dk, const unsigned short* dv, unsigned short* dqkv,
            float* partial, unsigned blocks, hipStream_t st) {
#define DPA_HEADS(N_, I_) hipLaunchKernelGGL((heads_bwd_kernel<L, N_, I_>), dim3(blocks), dim3(64 * WAVES), 0, st, a, dq, dk, dv, dqkv, partial)
    if (a.qw != nullptr) { if (a.interleaved) DPA_HEADS(true, true); else DPA_HEADS(true, false); }
    else { if (a.interleaved) DPA_HEADS(false, true); else DPA_HEADS(false, false); }
#undef DPA_HEADS
}

}  // namespace

int heads_partial_rows(long tokens) {
    const long b = (tokens + WAVES - 1) / WAVES;
    return (int)(b < 1 ? 1 : b > 1024 ? 1024 : b);
}

void heads_fwd(const HeadsArgs& a, void* q, void* k, hipStream_t st) {
    const long b = (a.tokens + WAVES - 1) / WAVES;
    const unsigned blocks = (unsigned)(b > 65536 ? 65536 : b);
    unsigned short *qp = (unsigned short*)q, *kp = (unsigned short*)k;
    if (a.D <= 32) fwd_of<4>(a, qp, kp, blocks, st);
    else if (a.D <= 64) fwd_of<8>(a, qp, kp, blocks, st);
    else if (a.D <= 128) fwd_of<16>(a, qp, kp, blocks, st);
    else fwd_of<32>(a, qp, kp, blocks, st);
}

void heads_bwd(const HeadsArgs& a, const void* dq, const void* dk, const void* dv, void* dqkv, float* partial, float* dqw, float* dkw, hipStream_t st) {
    const int blocks = heads_partial_rows(a.tokens);
    const unsigned short *q = (const unsigned short*)dq, *k = (const unsigned short*)dk, *v = (const unsigned short*)dv;
    unsigned short* o = (unsigned short*)dqkv;
    if (a.D <= 32) bwd_of<4>(a, q, k, v, o, partial, blocks, st);
    else if (a.D <= 64) bwd_of<8>(a, q, k, v, o, partial, blocks, st);
    else if (a.D <= 128) bwd_of<16>(a, q, k, v, o, partial, blocks, st);
    else bwd_of<32>(a, q, k, v, o, partial, blocks, st);
    if (a.qw != nullptr) reduce_partials2(partial, blocks, a.D, dqw, dkw, 0, st);
}

}  // namespace dpa
