// Rotary positions -- gfx950 (MI355X).
//
// A pair (a, b) of a head's channels turns by the angle t = position * inv_freq:
//   (a, b) -> A (a cos t - b sin t, b cos t + a sin t);    the gradient turns by -t with the same factor A.
// The first 2 * axes * pairs channels are `axes` sections, one a position axis (a token's row and column in an image grid, say); in a
// section of 2 P channels, pair p is (p, p + P) or, interleaved, (2 p, 2 p + 1).  Channels behind the sections are copied.
//
// Angles are 64-bit up to the fraction of a turn that is left (32 bits would be off by 0.06 rad at position 1e6); sine and cosine of that
// fraction are 32-bit.  The kernel is bound by HBM: x in, y out.  A thread holds the sines of VP pairs of one token and walks the heads
// with them, so the 64-bit part is paid once a token and not once a head; loads and stores are 16 bytes wide where P allows.
//
// 131072 tokens x 16 heads x 128 (64 turned) bf16: 239 us = 4.5 TB/s (a large copy: 4.7); 19200 x 8 x 32 fp32, two axes: 8.8 us = 4.5 TB/s;
// 16 tokens x 8 x 64: 3.6 us, a launch's latency.
#include "elem.h"

namespace {

using namespace dfsfm;

struct RotaryArgs {
    const void* x;
    int64_t xn, xl, xh;
    void* y;
    int64_t yn, yl, yh;
    const int64_t* pos;
    int64_t pn, pl, pa;
    const double* inv_freq;
    double turn;                // +-1 / 2 pi
    float amplitude;
    unsigned tokens, L, first;                // first: token of workgroup 0
    int H, D, pairs, axes, units, heads;      // units: threads a token; heads: heads a thread
};

template <typename T, int VP, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    constexpr int VC = 16 / sizeof(T);
    const unsigned per = 256u / a.units, sub = threadIdx.x / a.units;
    const unsigned tok = a.first + blockIdx.x * per + sub;
    if (sub >= per || tok >= a.tokens) return;
    const int unit = threadIdx.x % a.units, turned = a.axes * a.pairs / VP;
    const int64_t n = tok / a.L, l = tok % a.L;
    const int h0 = blockIdx.y * a.heads, h1 = min(a.H, h0 + a.heads);
    const T* x = static_cast<const T*>(a.x) + n * a.xn + l * a.xl + h0 * a.xh;
    T* y = static_cast<T*>(a.y) + n * a.yn + l * a.yl + h0 * a.yh;
    if (unit >= turned) {                                         // channels behind the sections
        const int c = 2 * a.axes * a.pairs + (unit - turned) * VC;
        for (int h = h0; h < h1; ++h, x += a.xh, y += a.yh) {
            float v[VC];                                          // fp32 holds every value of the three types
            load_f32<T, VC>(x + c, a.D - c, v);
            store_f32<T, VC>(y + c, a.D - c, v);
        }
        return;
    }
    const int axis = unit * VP / a.pairs, p = unit * VP % a.pairs;      // VP divides pairs: a thread stays in one section
    const double at = (double)a.pos[n * a.pn + l * a.pl + axis * a.pa] * a.turn;
    float co[VP], si[VP];
#pragma unroll
    for (int i = 0; i < VP; ++i) {
        double t = at * a.inv_freq[p + i];
        t -= rint(t);
        sincospif(2.f * (float)t, &si[i], &co[i]);
        si[i] *= a.amplitude;
        co[i] *= a.amplitude;
    }
    const int base = axis * 2 * a.pairs;
    if constexpr (INTERLEAVED) {
        x += base + 2 * p;
        y += base + 2 * p;
#pragma unroll 4
        for (int h = h0; h < h1; ++h, x += a.xh, y += a.yh) {
            float v[2 * VP], o[2 * VP];
            load_f32<T, 2 * VP>(x, v);
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                o[2 * i] = v[2 * i] * co[i] - v[2 * i + 1] * si[i];
                o[2 * i + 1] = v[2 * i + 1] * co[i] + v[2 * i] * si[i];
            }
            store_f32<T, 2 * VP>(y, 2 * VP, o);
        }
    } else {
        x += base + p;
        y += base + p;
#pragma unroll 4
        for (int h = h0; h < h1; ++h, x += a.xh, y += a.yh) {
            float u[VP], v[VP], o[VP], q[VP];
            load_f32<T, VP>(x, u);
            load_f32<T, VP>(x + a.pairs, v);
#pragma unroll
            for (int i = 0; i < VP; ++i) {
                o[i] = u[i] * co[i] - v[i] * si[i];
                q[i] = v[i] * co[i] + u[i] * si[i];
            }
            store_f32<T, VP>(y, VP, o);
            store_f32<T, VP>(y + a.pairs, VP, q);
        }
    }
}

template <typename T>
int rotary_launch(RotaryArgs a, bool interleaved, bool inplace, hipStream_t st) {
    constexpr int VC = 16 / sizeof(T);
    int vp = interleaved ? VC / 2 : VC;                           // 16 bytes a load
    while (a.pairs % vp) vp >>= 1;
    const int rest = a.D - 2 * a.axes * a.pairs;
    a.units = a.axes * a.pairs / vp + (inplace ? 0 : (rest + VC - 1) / VC);
    const unsigned per = 256u / a.units, bx = (a.tokens + per - 1) / per;
    // one thread a token and unit walks all heads where that leaves 2048 workgroups (eight a CU), fewer heads a thread otherwise
    const int slices = bx >= 2048 ? 1 : (int)((2048 + bx - 1) / bx);
    a.heads = (a.H + slices - 1) / slices;
    const dim3 blk(256);
    // a launch holds less than 2^32 threads along an axis: from 2^24 workgroups on (16.8 M tokens of 256 units) the tokens take several
    constexpr unsigned MOST = (1u << 24) - 1;
    for (unsigned b = 0; b < bx; b += MOST) {
        const dim3 grid(bx - b < MOST ? bx - b : MOST, (unsigned)((a.H + a.heads - 1) / a.heads));
        a.first = b * per;
#define DFSFM_ROT(VP_)                                                                                \
        if (vp == VP_) {                                                                              \
            if (interleaved)                                                                          \
                hipLaunchKernelGGL((rotary_kernel<T, VP_, true>), grid, blk, 0, st, a);               \
            else                                                                                      \
                hipLaunchKernelGGL((rotary_kernel<T, VP_, false>), grid, blk, 0, st, a);              \
        }
        DFSFM_ROT(1) DFSFM_ROT(2) DFSFM_ROT(4)
        if constexpr (VC == 8) DFSFM_ROT(8)
#undef DFSFM_ROT
    }
    return check_launch("dfsfm_rotary");
}

}  // namespace

extern "C" int dfsfm_rotary(const void* x, int64_t xn, int64_t xl, int64_t xh, void* y, int64_t yn, int64_t yl, int64_t yh,
                            const int64_t* positions, int64_t pn, int64_t pl, int64_t pa, const double* inv_freq, int pairs, int axes,
                            int interleaved, int backward, float amplitude, int N, int64_t L, int H, int D, int dtype, void* stream_) {
    if (N == 0 || L == 0 || H == 0) return DFSFM_OK;
    if (!x || !y || !positions || !inv_freq || N < 0 || L < 0 || H < 0 || D <= 0 || pairs <= 0 || axes <= 0) return DFSFM_E_BADARG;
    if ((int64_t)2 * pairs * axes > D) return DFSFM_E_BADARG;
    const bool inplace = x == y;
    if (inplace && (xn != yn || xl != yl || xh != yh)) return DFSFM_E_BADARG;
    // 512 channels are at most 256 threads a token; the heads' slices are a grid axis of 16 bits
    if (D > 512 || axes > 2 || H > 65535 || L > 0x7fffffff || (int64_t)N * L > 0x7fffffff) return DFSFM_E_UNSUPPORTED;
    RotaryArgs a{x, xn, xl, xh, y, yn, yl, yh, positions, pn, pl, pa, inv_freq, (backward ? -1.0 : 1.0) * 0.15915494309189535,
                 amplitude, (unsigned)(N * L), (unsigned)L, 0, H, D, pairs, axes, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream_);
    if (dtype == DFSFM_F32) return rotary_launch<float>(a, interleaved != 0, inplace, st);
    if (dtype == DFSFM_BF16) return rotary_launch<dfsfm::bf16>(a, interleaved != 0, inplace, st);
    if (dtype == DFSFM_F16) return rotary_launch<dfsfm::f16>(a, interleaved != 0, inplace, st);
    return DFSFM_E_UNSUPPORTED;
}
