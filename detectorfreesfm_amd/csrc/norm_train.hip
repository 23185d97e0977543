// Layer norm for training -- gfx950 (MI355X): the forward pass that keeps the rows' statistics, and its gradient.
//
//   forward   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), y = (x - m) r gamma + beta (+ residual)
//   backward  h = (x - m) r, g = dy gamma
//             dx = r (g - mean(g) - h mean(g h)),  dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both are bound by HBM: x (residual) in and y out, then x and dy in and dx out, each once.  A row lives in the registers of G lanes
// (NV vectors of 16 bytes each), so the mean, the squares around it and the result come from one read; G is the smallest power of two
// that holds the row with one vector a lane, the whole workgroup for wide rows.  Sums are 32-bit.  The weights' gradients are summed in
// registers over all rows a lane group sees, then over the workgroup's groups in LDS, then over the workgroups by a second kernel: every
// sum has a fixed order, no atomics.
//
// Time, kernels alone: 9600 x 256 fp32 forward with residual 6.4 us = 4.6 TB/s (a copy of 2 GB: 4.7); 450000 x 128 fp32 forward 123 and
// gradient 130 us = 5.6 and 5.3 TB/s (part of x comes from the last-level cache); 8192 x 4096 bf16 forward 26, gradient 42, weights' sums
// 5 us, 81 us a pass on inputs that are in no cache, where the five tensors of both take a copy 71.
#include "elem.h"

namespace {

using dfsfm::check_launch;
using dfsfm::load_f32;
using dfsfm::store_f32;
using dfsfm::Vec;

// Sum over the G lanes (a power of two up to 64, or the G threads of the workgroup) that share a row; every lane gets the same bits.
// `slot` alternates between calls so that one barrier a call is enough.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* lds, int& slot) {
#pragma unroll
    for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) v += __shfl_xor(v, o);
    if constexpr (G > 64) {
        float* part = lds + slot * (G / 64);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < G / 64; ++w) v += part[w];
        slot ^= 1;
    }
    return v;
}

// Threads of the workgroup that G lanes a row make.
constexpr int norm_threads(int G) { return G < 256 ? 256 : G; }

// How the vectors of a lane lie in a row of C elements.  EVEN: C is a multiple of V, a vector is whole or absent.  TAIL: the row's last
// vector is moved back to end with the row, so that it is one wide access too; `skip` of its first elements belong to the neighbour as well:
// they count in no sum, and both lanes store the same bits.  SHORT: C < V, element accesses of one lane.
enum Row { EVEN, TAIL, SHORT };

template <int V, int MODE>
struct Place {
    int c, skip;                                           // first column, elements that do not count (V: none does)
    __device__ __forceinline__ Place(int at, int C) {
        if constexpr (MODE == TAIL) {
            c = min(at, C - V);
            skip = min(at - c, V);
        } else {
            c = at < C ? at : 0;
            skip = at < C ? 0 : V;
        }
    }
    __device__ __forceinline__ bool counts(int e, int C) const {
        if constexpr (MODE == EVEN) return skip == 0;
        if constexpr (MODE == TAIL) return e >= skip;
        return skip == 0 && e < C;
    }
    template <typename T>
    __device__ __forceinline__ void load(const T* row, int C, float (&r)[V]) const {
        if constexpr (MODE == SHORT) {
            load_f32<T, V>(row, skip ? 0 : C, r);
        } else if constexpr (MODE == TAIL) {
            load_f32<T, V>(row + c, r);
        } else {
            if (skip == 0) {
                load_f32<T, V>(row + c, r);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) r[e] = 0.f;
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ typename Vec<T, V>::raw raw(const T* row, int C) const {
        typename Vec<T, V>::raw v;
        if constexpr (MODE == SHORT) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = skip == 0 && e < C ? row[e] : (T)0.f;
        } else if (MODE == TAIL || skip == 0) {
            v = *reinterpret_cast<const typename Vec<T, V>::type*>(row + c);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (T)0.f;
        }
        return v;
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, int C, const float (&r)[V]) const {
        if (skip < V) store_f32<T, V>(row + c, MODE == SHORT ? C : V, r);
    }
};

template <typename T, typename W, int G, int NV, int MODE>
__global__ __launch_bounds__(norm_threads(G)) void norm_forward_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ gamma,
                                                           const W* __restrict__ beta, float eps, const T* __restrict__ residual,
                                                           int64_t ldr, T* __restrict__ y, float* __restrict__ mean,
                                                           float* __restrict__ rstd, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T), RPB = norm_threads(G) / G;
    constexpr bool KEEP = NV * V <= 8;                     // gamma and beta stay in registers over the rows
    __shared__ float lds[G > 64 ? G / 32 : 1];
    int slot = 0;
    const int lane = threadIdx.x % G, sub = threadIdx.x / G;
    float ga[KEEP ? NV : 1][V], be[KEEP ? NV : 1][V];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
            at.load(gamma, C, ga[i]);
            at.load(beta, C, be[i]);
        }
    }
    const float inv = 1.f / (float)C;
    // G > 64: the barriers inside row_sum need every thread of the workgroup, and with RPB = 1 all of them share the row
    for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < rows; row += (int64_t)gridDim.x * RPB) {
        float v[NV][V], s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
            at.load(x + row * ldx, C, v[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += MODE != TAIL || at.counts(e, C) ? v[i][e] : 0.f;
        }
        const float m = row_sum<G>(s, lds, slot) * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= m;
                s += at.counts(e, C) ? v[i][e] * v[i][e] : 0.f;
            }
        }
        const float r = 1.f / sqrtf(row_sum<G>(s, lds, slot) * inv + eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
            if constexpr (!KEEP) {
                at.load(gamma, C, ga[0]);
                at.load(beta, C, be[0]);
            }
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(v[i][e] * r, ga[KEEP ? i : 0][e], be[KEEP ? i : 0][e]);
            if (residual) {
                float q[V];
                at.load(residual + row * ldr, C, q);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] += q[e];
            }
            at.store(y + row * C, C, o);
        }
        if (lane == 0) {
            mean[row] = m;
            rstd[row] = r;
        }
    }
}

// part: [gridDim.x][2][C] sums of the workgroups, or null when the launch has one workgroup, which then writes the gradients itself.
template <typename T, typename W, int G, int NV, int MODE>
__global__ __launch_bounds__(norm_threads(G)) void norm_backward_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            const W* __restrict__ gamma, T* __restrict__ dx, W* __restrict__ dgamma,
                                                            W* __restrict__ dbeta, float* __restrict__ part, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T), RPB = norm_threads(G) / G;
    __shared__ float lds[G > 64 ? G / 32 : 1];
    __shared__ float sums[RPB > 1 ? 256 * V * NV : 1];
    int slot = 0;
    const int lane = threadIdx.x % G, sub = threadIdx.x / G;
    float ga[NV][V], sg[NV][V], sb[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Place<V, MODE> at((i * G + lane) * V, C);
        at.load(gamma, C, ga[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) sg[i][e] = sb[i][e] = 0.f;
    }
    const float inv = 1.f / (float)C;
    const int64_t first = (int64_t)blockIdx.x * RPB + sub, step = (int64_t)gridDim.x * RPB;
    typename Vec<T, V>::raw nx[NV], ny[NV];                // the next row, on its way while this one is summed
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](int64_t row) {
        nm = mean[row];
        nr = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
            nx[i] = at.raw(x + row * ldx, C);
            ny[i] = at.raw(dy + row * lddy, C);
        }
    };
    if (first < rows) fetch(first);
    for (int64_t row = first; row < rows; row += step) {
        const float m = nm, r = nr;
        float h[NV][V], g[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[i][e] = (float)nx[i][e];
                g[i][e] = (float)ny[i][e];
            }
        if (row + step < rows) fetch(row + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[i][e] = (h[i][e] - m) * r;               // an absent vector's g is 0: its h counts for nothing
                const float d = MODE != TAIL || at.counts(e, C) ? g[i][e] : 0.f;
                sb[i][e] += d;
                sg[i][e] = fmaf(d, h[i][e], sg[i][e]);
                const float w = d * ga[i][e];
                s1 += w;
                s2 = fmaf(w, h[i][e], s2);
            }
        }
        const float c1 = row_sum<G>(s1, lds, slot) * inv, c2 = row_sum<G>(s2, lds, slot) * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = r * (g[i][e] * ga[i][e] - c1 - h[i][e] * c2);
            at.store(dx + row * C, C, o);
        }
    }
    if (!dgamma) return;
    if constexpr (RPB > 1) {                               // the workgroup's groups, in their order
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const Place<V, MODE> at((i * G + lane) * V, C);
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at.counts(e, C)) sums[sub * NV * G * V + at.c + e] = k ? sb[i][e] : sg[i][e];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += 256) {
                float s = 0.f;
                for (int u = 0; u < RPB; ++u) s += sums[u * NV * G * V + c];
                if (part)
                    part[((int64_t)blockIdx.x * 2 + k) * C + c] = s;
                else
                    (k ? dbeta : dgamma)[c] = (W)s;
            }
        }
    } else {
        float* pg = part ? part + (int64_t)blockIdx.x * 2 * C : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Place<V, MODE> at((i * G + lane) * V, C);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (at.counts(e, C)) {
                    if (pg) {
                        pg[at.c + e] = sg[i][e];
                        pg[C + at.c + e] = sb[i][e];
                    } else {
                        dgamma[at.c + e] = (W)sg[i][e];
                        dbeta[at.c + e] = (W)sb[i][e];
                    }
                }
        }
    }
}

// dgamma | dbeta = sum over P workgroups of part [P][2 C]: 32 columns x 32 slices of the workgroups a block, slices joined in LDS.
template <typename W>
__global__ __launch_bounds__(1024) void norm_weights_kernel(const float* __restrict__ part, int P, W* __restrict__ dgamma,
                                                            W* __restrict__ dbeta, int C) {
    __shared__ float sums[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col, C2 = 2 * (int64_t)C;
    float s = 0.f;
    if (c < C2)
#pragma unroll 8
        for (int p = slice; p < P; p += 32) s += part[p * C2 + c];
    sums[slice][col] = s;
    __syncthreads();
    if (slice == 0 && c < C2) {
        s = 0.f;
#pragma unroll
        for (int u = 0; u < 32; ++u) s += sums[u][col];
        if (c < C)
            dgamma[c] = (W)s;
        else
            dbeta[c - C] = (W)s;
    }
}

constexpr int NORM_MAX_C = 16384;

// Lanes and vectors a lane that hold a row of C elements, V a vector.
struct Split {
    int G, NV;
};
Split split_row(int C, int V) {
    const int n = (C + V - 1) / V;
    int g = 4, nv = 1;
    if (n <= 128) {                                        // lanes of one wave, two vectors each at most
        while (g < n && g < 64) g <<= 1;
    } else {                                               // 16 elements a thread at most: the gradient holds five values for each
        g = n <= 256 * 16 / V ? 256 : 1024;
    }
    while (g * nv < n) nv <<= 1;
    return {g, nv};
}

// The instance of a row split (every G, NV that split_row gives for C up to NORM_MAX_C) and of C's rest.
#define DFSFM_NORM_CASE(K, G_, NV_)           \
    if (C >= V && s.G == G_ && s.NV == NV_) { \
        if (C % V == 0) K(G_, NV_, EVEN);     \
        else K(G_, NV_, TAIL);                \
    }
#define DFSFM_NORM_PICK(K)                                                                                                              \
    if (C < V) K(4, 1, SHORT);                                                                                                          \
    DFSFM_NORM_CASE(K, 4, 1) DFSFM_NORM_CASE(K, 8, 1) DFSFM_NORM_CASE(K, 16, 1) DFSFM_NORM_CASE(K, 32, 1) DFSFM_NORM_CASE(K, 64, 1)      \
    DFSFM_NORM_CASE(K, 64, 2) DFSFM_NORM_CASE(K, 256, 1) DFSFM_NORM_CASE(K, 256, 2) DFSFM_NORM_CASE(K, 1024, 2)                          \
    if constexpr (V == 4) {                                                                                                             \
        DFSFM_NORM_CASE(K, 256, 4) DFSFM_NORM_CASE(K, 1024, 4)                                                                          \
    } else {                                                                                                                            \
        DFSFM_NORM_CASE(K, 1024, 1)                                                                                                     \
    }

int norm_blocks_backward(int64_t rows, int C, int V) {
    const Split s = split_row(C, V);
    const int rpb = norm_threads(s.G) / s.G;
    // Eight rows a group at least and 512 workgroups at most, so that the partial sums stay small next to the rows: 8192 x 4096 bf16 forward
    // and gradient 83 us, 95 with 1024 workgroups, whose sums are a quarter of all bytes.
    const int64_t want = (rows + rpb * 8 - 1) / (rpb * 8);
    return (int)(want < 512 ? (want < 1 ? 1 : want) : 512);
}

template <typename T, typename W>
int forward_launch(const void* x, int64_t ldx, const void* gamma, const void* beta, float eps, const void* residual, int64_t ldr, void* y,
                   float* mean, float* rstd, int64_t rows, int C, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const Split s = split_row(C, V);
    const int rpb = norm_threads(s.G) / s.G;
    const int64_t want = (rows + rpb - 1) / rpb;
    const dim3 grid((unsigned)(want < 4096 ? want : 4096)), blk(norm_threads(s.G));
#define DFSFM_NORM_F(G_, NV_, MODE_)                                                                                                  \
    hipLaunchKernelGGL((norm_forward_kernel<T, W, G_, NV_, MODE_>), grid, blk, 0, st, (const T*)x, ldx, (const W*)gamma,              \
                       (const W*)beta, eps, (const T*)residual, ldr, (T*)y, mean, rstd, rows, C)
    DFSFM_NORM_PICK(DFSFM_NORM_F)
#undef DFSFM_NORM_F
    return check_launch("dfsfm_layernorm_forward");
}

template <typename T, typename W>
int backward_launch(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* mean, const float* rstd, const void* gamma,
                    void* dx, void* dgamma, void* dbeta, int64_t rows, int C, float* part, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const Split s = split_row(C, V);
    const int P = norm_blocks_backward(rows, C, V);
    if (P == 1) part = nullptr;
    const dim3 grid((unsigned)P), blk(norm_threads(s.G));
#define DFSFM_NORM_B(G_, NV_, MODE_)                                                                                                   \
    hipLaunchKernelGGL((norm_backward_kernel<T, W, G_, NV_, MODE_>), grid, blk, 0, st, (const T*)dy, lddy, (const T*)x, ldx, mean,     \
                       rstd, (const W*)gamma, (T*)dx, (W*)dgamma, (W*)dbeta, part, rows, C)
    DFSFM_NORM_PICK(DFSFM_NORM_B)
#undef DFSFM_NORM_B
    if (dgamma && part)
        hipLaunchKernelGGL((norm_weights_kernel<W>), dim3((unsigned)((2 * C + 31) / 32)), dim3(1024), 0, st, part, P, (W*)dgamma, (W*)dbeta, C);
    return check_launch("dfsfm_layernorm_backward");
}

#undef DFSFM_NORM_PICK
}  // namespace

extern "C" int dfsfm_layernorm_forward(const void* x, int64_t ldx, const void* gamma, const void* beta, int wtype, float eps,
                                       const void* residual, int64_t ldr, void* y, float* mean, float* rstd, int64_t rows, int C, int dtype,
                                       void* stream_) {
    if (rows == 0) return DFSFM_OK;
    if (!x || !gamma || !beta || !y || !mean || !rstd || rows < 0 || C <= 0 || ldx < 0 || (residual && ldr < 0)) return DFSFM_E_BADARG;
    if (C > NORM_MAX_C || (wtype != dtype && wtype != DFSFM_F32)) return DFSFM_E_UNSUPPORTED;
    hipStream_t st = static_cast<hipStream_t>(stream_);
#define DFSFM_ARGS x, ldx, gamma, beta, eps, residual, ldr, y, mean, rstd, rows, C, st
    if (dtype == DFSFM_F32) return forward_launch<float, float>(DFSFM_ARGS);
    if (dtype == DFSFM_BF16) return wtype == DFSFM_F32 ? forward_launch<dfsfm::bf16, float>(DFSFM_ARGS) : forward_launch<dfsfm::bf16, dfsfm::bf16>(DFSFM_ARGS);
    if (dtype == DFSFM_F16) return wtype == DFSFM_F32 ? forward_launch<dfsfm::f16, float>(DFSFM_ARGS) : forward_launch<dfsfm::f16, dfsfm::f16>(DFSFM_ARGS);
#undef DFSFM_ARGS
    return DFSFM_E_UNSUPPORTED;
}

extern "C" size_t dfsfm_layernorm_backward_workspace(int64_t rows, int C, int dtype) {
    if (rows <= 0 || C <= 0 || C > NORM_MAX_C || dtype < DFSFM_F32 || dtype > DFSFM_F16) return 0;
    return (size_t)norm_blocks_backward(rows, C, dtype == DFSFM_F32 ? 4 : 8) * 2 * C * sizeof(float);
}

extern "C" int dfsfm_layernorm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* mean, const float* rstd,
                                        const void* gamma, int wtype, void* dx, void* dgamma, void* dbeta, int64_t rows, int C, int dtype,
                                        void* workspace, size_t workspace_bytes, void* stream_) {
    hipStream_t st = static_cast<hipStream_t>(stream_);
    if (rows < 0 || C <= 0 || (dgamma == nullptr) != (dbeta == nullptr)) return DFSFM_E_BADARG;
    if (C > NORM_MAX_C || dtype < DFSFM_F32 || dtype > DFSFM_F16 || (wtype != dtype && wtype != DFSFM_F32)) return DFSFM_E_UNSUPPORTED;
    if (rows == 0) {                                       // sums over no rows are zeros
        if (!dgamma) return DFSFM_OK;
        const dim3 grid((unsigned)((2 * C + 31) / 32)), blk(1024);
        if (wtype == DFSFM_F32)
            hipLaunchKernelGGL((norm_weights_kernel<float>), grid, blk, 0, st, nullptr, 0, (float*)dgamma, (float*)dbeta, C);
        else if (wtype == DFSFM_BF16)
            hipLaunchKernelGGL((norm_weights_kernel<dfsfm::bf16>), grid, blk, 0, st, nullptr, 0, (dfsfm::bf16*)dgamma, (dfsfm::bf16*)dbeta, C);
        else
            hipLaunchKernelGGL((norm_weights_kernel<dfsfm::f16>), grid, blk, 0, st, nullptr, 0, (dfsfm::f16*)dgamma, (dfsfm::f16*)dbeta, C);
        return dfsfm::check_launch("dfsfm_layernorm_backward");
    }
    if (!dy || !x || !mean || !rstd || !gamma || !dx || ldx < 0 || lddy < 0) return DFSFM_E_BADARG;
    if (dgamma && (!workspace || workspace_bytes < dfsfm_layernorm_backward_workspace(rows, C, dtype))) return DFSFM_E_WORKSPACE;
    float* part = dgamma ? static_cast<float*>(workspace) : nullptr;
#define DFSFM_ARGS dy, lddy, x, ldx, mean, rstd, gamma, dx, dgamma, dbeta, rows, C, part, st
    if (dtype == DFSFM_F32) return backward_launch<float, float>(DFSFM_ARGS);
    if (dtype == DFSFM_BF16) return wtype == DFSFM_F32 ? backward_launch<dfsfm::bf16, float>(DFSFM_ARGS) : backward_launch<dfsfm::bf16, dfsfm::bf16>(DFSFM_ARGS);
    return wtype == DFSFM_F32 ? backward_launch<dfsfm::f16, float>(DFSFM_ARGS) : backward_launch<dfsfm::f16, dfsfm::f16>(DFSFM_ARGS);
#undef DFSFM_ARGS
}
