// Softmax cross attention with its gradient -- gfx950 (MI355X).
//
//   forward   s = scale q k^T over the keys that are there, p = softmax(s), out = p v, lse = log sum exp(s); no key: out = 0, lse = -inf
//   backward  delta = <dout, out>, ds = p (dout v^T - delta), dq = scale ds k, dk = scale ds^T q, dv = p^T dout
//
// All products run on 32 x 32 MFMA tiles with 32-bit accumulators; fp32 tensors use the 32-bit matrix instruction (no split, no loss of
// range), bf16 and fp16 the 16-bit one.  A lane holds ONE column of the score tile: a query in the forward and dq kernels, a key in the
// dk / dv kernel, so the running maximum, the sum and the scale of a query are per-lane values, and the accumulator registers of a score
// tile are, in their order, the operand of the next product (its other operand is read from LDS with the same order of the inner index):
// the scores never leave the registers.  The query heads that share a key head are rows of one problem: row r is (query r / G, head r % G).
//
// Keys that are not there (behind kv_lens, or where kv_mask is 0) are zeroed on their way into LDS and get a bias of -inf, whatever the
// memory held; a tile without any is skipped.  Few rows: the keys (or, for dk / dv, the rows) are cut into splits that write 32-bit partial
// results, joined in a fixed order by a second kernel.  No atomics.
#include "elem.h"

namespace {

using dfsfm::bf16;
using dfsfm::f16;
using dfsfm::check_launch;
using dfsfm::mfma32_row;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KT = 64;                     // rows of a staged tile
constexpr float NEG = -INFINITY;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// Operands of a 32 x 32 x 16 product: lane (i = lane & 31, h = lane >> 5) holds row i, inner indices 8 h .. 8 h + 7.
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16> {
    typedef f16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {
    typedef f32x8 frag;
    static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

template <typename T>
using Frag = typename Mma<T>::frag;

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)0.f;
    return f;
}

// 8 consecutive channels from global memory (any alignment)
template <typename T>
__device__ __forceinline__ Frag<T> load8(const T* p) {
    typedef typename dfsfm::Vec<T, 8>::type vec;
    return *reinterpret_cast<const vec*>(p);
}

// Row pitches of a tile in LDS, in elements.  Rows read as A operands (16 bytes a lane, a row a lane): pitch = DP + 16 bytes.  Rows read
// transposed (four rows x 32 bytes by 16 lanes): DP + 32 bytes.  Both spread the lanes of a cycle over all banks.
template <typename T, int DP>
constexpr int PITCH = DP + 16 / sizeof(T);
template <typename T, int DP>
constexpr int PITCH_T = DP + 32 / sizeof(T);

// A operand: rows row .. row + 31 of a tile, inner index = channels col .. col + 15.
template <typename T>
__device__ __forceinline__ Frag<T> read_rows(const T* tile, int pitch, int row, int col, int lane) {
    typedef Frag<T> at16 __attribute__((aligned(16)));                    // pitches are multiples of 16 bytes, not of 32
    return *reinterpret_cast<const at16*>(tile + (row + (lane & 31)) * pitch + col + 8 * (lane >> 5));
}

// A operand of the transposed tile: rows = channels col .. col + 31, inner index = tile rows in the order of an accumulator's registers:
// slot j of half h is row + (j & 3) + 8 (j >> 2) + 4 h.
template <typename T>
__device__ __forceinline__ Frag<T> read_cols(const T* tile, int pitch, int row, int col, int lane) {
    if constexpr (sizeof(T) == 2) {
        // 16 lanes read a 4 x 16 block, 8 bytes each along its rows; the transposed read hands lane i the block's column i
        const int i = lane & 15;
        const T* p = tile + (row + 4 * (lane >> 5) + (i >> 2)) * pitch + col + (lane & 16) + 4 * (i & 3);
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * pitch));
        const auto v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(Frag<T>, v);
    } else {
        Frag<T> f;
        const T* p = tile + (row + 4 * (lane >> 5)) * pitch + col + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = p[((j & 3) + 8 * (j >> 2)) * pitch];
        return f;
    }
}

// Registers 8 t .. 8 t + 7 of a score tile as the other operand (round to nearest even).
template <typename T>
__device__ __forceinline__ Frag<T> pack8(const f32x16& s, int t) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)s[8 * t + j];
    return f;
}

// Waves a SIMD that the forward and dq kernels are compiled for: two (256 registers a wave), so that one wave's exponentials run beside the
// other's products.  fp32 at D = 128 holds twice the operands and would spill.
template <typename T, int DP>
constexpr int WAVES = sizeof(T) == 4 && DP == 128 ? 1 : 2;

struct Tensor {
    const void* p;
    int64_t n, l, h;                       // element strides of [N, length, heads, D]; the channel stride is 1
};

struct Attn {
    Tensor q, k, v, dout, out;
    const int* lens;
    const uint8_t* mask;                   // [N, S]
    void* o[2];                            // results (out, or dq, or dk and dv): dense, in T or, with splits, 32-bit partials
    float* lse;                            // [N, H, L]
    float* ml;                             // forward partials: maximum, sum [splits][N, H, L][2]
    float* delta;                          // [N, H, L]
    int64_t numel;                         // elements of one partial result
    int N, L, S, H, G, D, splits, tiles;
    float scale;
};

// What a workgroup works on: grid.x = (splits, N * kv heads, tiles), tiles fastest: neighbours in time are tiles of one head, spread over all
// XCDs, so sequences of unequal lengths load the chip evenly.  Heads fastest (a head's tiles on one XCD's L2) left XCDs with short sequences
// idle: 1.11 ms against 0.82 for the forward pass of 4 x 4800 x 6400 (ragged) x 16 heads x 128.
struct Job {
    int n, hk, tile, split;
    __device__ __forceinline__ Job(const Attn& a) {
        const int hkv = a.H / a.G, heads = a.N * hkv;
        tile = blockIdx.x % a.tiles;
        const int rest = blockIdx.x / a.tiles, head = rest % heads;
        split = rest / heads;
        n = head / hkv;
        hk = head % hkv;
    }
};

__device__ __forceinline__ int valid_len(const Attn& a, int n) { return a.lens ? min(max(a.lens[n], 0), a.S) : a.S; }

// A tile of 64 rows x DP channels on its way from memory through the registers of 256 threads into LDS.  A thread's 32-bit byte offsets
// within a tile are the same for every whole tile: the address costs one scalar base a tile and no vector arithmetic.
template <typename T, int DP>
struct Stage {
    static constexpr int VPR = DP / 8, PER = KT * VPR / 256;
    Frag<T> r[PER];
    unsigned off[PER];
    unsigned stride;                       // bytes a row
    int D;
    __device__ __forceinline__ Stage(int64_t stride_, int D_) : stride((unsigned)(stride_ * sizeof(T))), D(D_) {
#pragma unroll
        for (int i = 0; i < PER; ++i) off[i] = offset(i, KT - 1);
    }
    __device__ __forceinline__ unsigned offset(int i, int last) const {
        const int e = threadIdx.x + 256 * i;
        return min(e / VPR, last) * stride + e % VPR * 8 * (unsigned)sizeof(T);
    }
    // rows base .. base + rows - 1, the last one again behind them
    __device__ __forceinline__ void load(const T* base, int rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned o = rows >= KT ? off[i] : offset(i, rows - 1);
            const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + o);
            r[i] = (threadIdx.x + 256 * i) % VPR * 8 < D ? load8<T>(p) : zero_frag<T>();
        }
    }
    // rows whose bit in `keep` is 0 become zeros
    __device__ __forceinline__ void store(T* tile, int pitch, unsigned long long keep) const {
        typedef Frag<T> at16 __attribute__((aligned(16)));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = threadIdx.x + 256 * i, row = e / VPR, c = e % VPR * 8;
            *reinterpret_cast<at16*>(tile + row * pitch + c) = ~keep == 0 || keep >> row & 1 ? r[i] : zero_frag<T>();
        }
    }
};

// Bits of the keys s0 .. s0 + 63 that are there; the same in every wave.
__device__ __forceinline__ unsigned long long key_bits(const Attn& a, int n, int s0, int end) {
    const int s = s0 + (threadIdx.x & 63);
    bool ok = s < end;
    if (a.mask) ok = ok && a.mask[(int64_t)n * a.S + min(s, a.S - 1)] != 0;
    return __ballot(ok);
}

__device__ __forceinline__ f32x16 splat16(float x) {
    f32x16 v;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = x;
    return v;
}

// 16 values of a 32-row vector in LDS in the order of an accumulator's registers
__device__ __forceinline__ f32x16 rows16(const float* v, int lane) {
    f32x16 r;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(v + 8 * g + 4 * (lane >> 5));
#pragma unroll
        for (int e = 0; e < 4; ++e) r[4 * g + e] = t[e];
    }
    return r;
}

// out is a mean of values of v, but its weights are rounded and their sum is not: with v at fp16's largest value the quotient can pass it by
// 2^-11 and would round to infinity.  A value that close behind the range becomes the largest one; infinities in v stay.
template <typename T>
__device__ __forceinline__ float within_range(float x) {
    if constexpr (__is_same(T, f16)) return fabsf(x) < 65600.f ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
    return x;
}

// Stores a transposed accumulator (channels x columns) to the dense row of this lane's column.
template <typename T, int DB, bool MEAN = false>
__device__ __forceinline__ void store_col(T* row, const f32x16 (&acc)[DB], float f, int D, int lane) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * b + 8 * g + 4 * (lane >> 5);
            if (d < D) {                    // D is a multiple of 8
                float t[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = MEAN ? within_range<T>(acc[b][4 * g + e] * f) : acc[b][4 * g + e] * f;
                dfsfm::store_f32<T, 4>(row + d, 4, t);
            }
        }
}

// The operand of a fp16 product whose factors may be far below 1 (p times a gradient): a power of two per column, taken from the largest
// value so far, keeps the values between 2^-14 and 2^15 without changing a bit of them; the accumulator follows it.  The other types have
// fp32's range and need none.
template <typename T, int DB>
struct ColumnScale {
    float f = 1.f, seen = 0.f;
    template <int NB>
    __device__ __forceinline__ void apply(f32x16 (&ds)[NB], f32x16 (&acc)[DB]) {
        if constexpr (sizeof(T) == 2 && !__is_same(T, bf16)) {
            float m = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(ds[b][j]));
            m = fmaxf(m, dfsfm::from_xor32(m, threadIdx.x & 63));
            if (__ballot(m > seen)) {
                if (m > seen) {
                    // 2^11 leaves room for values 8 times larger before the next step; exponents stay those of normal numbers
                    const float old = f;
                    const int e = min(max(138 - (int)(__float_as_uint(m) >> 23), -100), 100);
                    if (m < INFINITY) f = __uint_as_float((unsigned)(e + 127) << 23);
                    seen = m * 8.f;
                    const float c = f / old;
#pragma unroll
                    for (int b = 0; b < DB; ++b)
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[b][j] *= c;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) ds[b][j] *= f;
        }
    }
};

// ---------------------------------------------------------------- forward
// 4 waves x 32 rows a workgroup; tiles of 64 keys, two in LDS.
template <typename T, int DP>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void attn_forward_kernel(const Attn a) {
    constexpr int KP = PITCH<T, DP>, VP = PITCH_T<T, DP>, DB = DP / 32, KS = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* ks = reinterpret_cast<T*>(smem);
    T* vs = ks + 2 * KT * KP;
    float* bias = reinterpret_cast<float*>(vs + 2 * KT * VP);            // [2][64]
    const Job job(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int R = a.L * a.G, r = job.tile * 128 + wave * 32 + (lane & 31);
    const int l = r / a.G, h = job.hk * a.G + r % a.G;
    const int len = valid_len(a, job.n);
    const int per = ((len + KT - 1) / KT + a.splits - 1) / a.splits * KT;   // keys a split, whole tiles
    const int beg = min(len, job.split * per), end = min(len, beg + per);

    Frag<T> qf[KS];
    const T* qp = static_cast<const T*>(a.q.p) + job.n * a.q.n + (int64_t)min(l, a.L - 1) * a.q.l + h * a.q.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * (lane >> 5);
        qf[s] = r < R && c < a.D ? load8<T>(qp + c) : zero_frag<T>();
    }
    const T* kb = static_cast<const T*>(a.k.p) + job.n * a.k.n + job.hk * a.k.h;
    const T* vb = static_cast<const T*>(a.v.p) + job.n * a.v.n + job.hk * a.v.h;
    Stage<T, DP> sk(a.k.l, a.D), sv(a.v.l, a.D);
    auto fetch = [&](int s0) {
        sk.load(kb + s0 * a.k.l, end - s0);
        sv.load(vb + s0 * a.v.l, end - s0);
    };
    f32x16 acc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) acc[b] = splat16(0.f);
    float m = NEG, sum = 0.f;               // maximum of scale * log2(e) * q k, sum of this lane's half of the keys
    const float c = a.scale * LOG2E;
    if (beg < end) fetch(beg);
    int buf = 0;
    for (int s0 = beg; s0 < end; s0 += KT, buf ^= 1) {
        const unsigned long long bits = key_bits(a, job.n, s0, end);
        T* kt = ks + buf * KT * KP;
        T* vt = vs + buf * KT * VP;
        float* bt = bias + buf * KT;
        sk.store(kt, KP, bits);
        sv.store(vt, VP, bits);
        if (threadIdx.x < KT) bt[threadIdx.x] = bits >> threadIdx.x & 1 ? 0.f : NEG;
        __syncthreads();                    // the other buffer's readers passed the barrier before this tile's writers came here
        if (s0 + KT < end) fetch(s0 + KT);
        if (bits == 0) continue;
        f32x16 st[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            st[b] = ~bits ? rows16(bt + 32 * b, lane) : splat16(0.f);
#pragma unroll
            for (int s = 0; s < KS; ++s) st[b] = Mma<T>::run(read_rows(kt, KP, 32 * b, 16 * s, lane), qf[s], st[b]);
        }
        float t = NEG;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) t = fmaxf(t, st[b][j]);
        t = fmaxf(t, dfsfm::from_xor32(t, lane)) * c;
        if (__ballot(t > m)) {
            const float mn = fmaxf(m, t), f = m == NEG ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[b][j] *= f;
        }
        const float mm = m == NEG ? 0.f : m;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                st[b][j] = __builtin_amdgcn_exp2f(fmaf(st[b][j], c, -mm));
                sum += st[b][j];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> p = pack8<T>(st[b], u);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = Mma<T>::run(read_cols(vt, VP, 32 * b + 16 * u, 32 * d, lane), p, acc[d]);
            }
        }
    }
    sum = dfsfm::add_xor32(sum);
    if (r >= R) return;
    const int64_t row = ((int64_t)job.n * a.L + l) * a.H + h, at = ((int64_t)job.n * a.H + h) * a.L + l;
    if (a.splits > 1) {
        store_col<float, DB>(static_cast<float*>(a.o[0]) + job.split * a.numel + row * a.D, acc, 1.f, a.D, lane);
        if (lane < 32) {
            float* ml = a.ml + ((int64_t)job.split * a.N * a.H * a.L + at) * 2;
            ml[0] = m;
            ml[1] = sum;
        }
    } else {
        store_col<T, DB, true>(static_cast<T*>(a.o[0]) + row * a.D, acc, sum > 0.f || sum != sum ? 1.f / sum : 0.f, a.D, lane);
        if (lane < 32) a.lse[at] = fmaf(m == NEG ? 0.f : m, LN2, logf(sum));
    }
}

// Joins the forward partials: 8 lanes x 4 channels a step, a row each 8 lanes.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const Attn a) {
    const int64_t rows = (int64_t)a.N * a.L * a.H, row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (row >= rows) return;
    const int h = (int)(row % a.H);
    const int64_t nl = row / a.H, at = (nl / a.L * a.H + h) * a.L + nl % a.L;
    float m = NEG, sum = 0.f;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.ml[(s * rows + at) * 2]);
    const float mm = m == NEG ? 0.f : m;
    for (int s = 0; s < a.splits; ++s) sum += a.ml[(s * rows + at) * 2 + 1] * __builtin_amdgcn_exp2f(a.ml[(s * rows + at) * 2] - mm);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    for (int d = (threadIdx.x & 7) * 4; d < a.D; d += 32) {
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f(a.ml[(s * rows + at) * 2] - mm) * inv;
            float t[4];
            dfsfm::load_f32<float, 4>(static_cast<const float*>(a.o[0]) + s * a.numel + row * a.D + d, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(t[e], f, o[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = within_range<T>(o[e]);
        dfsfm::store_f32<T, 4>(static_cast<T*>(a.o[1]) + row * a.D + d, 4, o);
    }
    if ((threadIdx.x & 7) == 0) a.lse[at] = fmaf(mm, LN2, logf(sum));
}

// ---------------------------------------------------------------- backward
// delta[n, h, l] = <dout, out> in 32 bits: 8 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(const Attn a) {
    const int64_t rows = (int64_t)a.N * a.L * a.H, row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (row >= rows) return;
    const int h = (int)(row % a.H);
    const int64_t nl = row / a.H, n = nl / a.L, l = nl % a.L;
    const T* x = static_cast<const T*>(a.dout.p) + n * a.dout.n + l * a.dout.l + h * a.dout.h;
    const T* y = static_cast<const T*>(a.out.p) + n * a.out.n + l * a.out.l + h * a.out.h;
    float s = 0.f;
    for (int d = (threadIdx.x & 7) * 8; d < a.D; d += 64) {
        float u[8], v[8];
        dfsfm::load_f32<T, 8>(x + d, u);
        dfsfm::load_f32<T, 8>(y + d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(u[e], v[e], s);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 7) == 0) a.delta[(n * a.H + h) * a.L + l] = s;
}

// dq: the forward kernel's frame, K read both ways.
//
// SHORT (up to 128 keys: both tiles stay in LDS) also computes delta, as the sum of p dp over the keys it is equal to.  The sum over the
// channels of dout times the ROUNDED out is off by half a step of out, an error that all keys of a row share: over many keys it drowns in
// the roundings of ds, over few it does not (dq of 4800 x 77 fp16: 3.2e-4 off in the 2-norm against 2.1e-4 that the output's rounding alone
// costs).  Two of three products are then made twice, over two tiles at most; a pass over dout and out is saved.
template <typename T, int DP, bool SHORT>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void attn_dq_kernel(const Attn a) {
    constexpr int KP = PITCH_T<T, DP>, VP = PITCH<T, DP>, DB = DP / 32, KS = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* ks = reinterpret_cast<T*>(smem);
    T* vs = ks + 2 * KT * KP;
    float* bias = reinterpret_cast<float*>(vs + 2 * KT * VP);
    const Job job(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int R = a.L * a.G, r = job.tile * 128 + wave * 32 + (lane & 31);
    const int l = r / a.G, h = job.hk * a.G + r % a.G;
    const int len = valid_len(a, job.n);
    const int per = ((len + KT - 1) / KT + a.splits - 1) / a.splits * KT;
    const int beg = min(len, job.split * per), end = min(len, beg + per);

    Frag<T> qf[KS], of[KS];
    const T* qp = static_cast<const T*>(a.q.p) + job.n * a.q.n + (int64_t)min(l, a.L - 1) * a.q.l + h * a.q.h;
    const T* op = static_cast<const T*>(a.dout.p) + job.n * a.dout.n + (int64_t)min(l, a.L - 1) * a.dout.l + h * a.dout.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * (lane >> 5);
        qf[s] = r < R && c < a.D ? load8<T>(qp + c) : zero_frag<T>();
        of[s] = r < R && c < a.D ? load8<T>(op + c) : zero_frag<T>();
    }
    const int64_t at = ((int64_t)job.n * a.H + h) * a.L + l;
    const float c = a.scale * LOG2E, lse = r < R ? a.lse[at] : NEG;
    const float lse2 = lse == NEG ? INFINITY : lse * LOG2E;              // a row without keys has p = 0
    float delta = !SHORT && r < R ? a.delta[at] : 0.f;
    const T* kb = static_cast<const T*>(a.k.p) + job.n * a.k.n + job.hk * a.k.h;
    const T* vb = static_cast<const T*>(a.v.p) + job.n * a.v.n + job.hk * a.v.h;
    Stage<T, DP> sk(a.k.l, a.D), sv(a.v.l, a.D);
    auto fetch = [&](int s0) {
        sk.load(kb + s0 * a.k.l, end - s0);
        sv.load(vb + s0 * a.v.l, end - s0);
    };
    auto stage = [&](int s0, int buf) {
        const unsigned long long bits = key_bits(a, job.n, s0, end);
        sk.store(ks + buf * KT * KP, KP, bits);
        sv.store(vs + buf * KT * VP, VP, bits);
        if (threadIdx.x < KT) bias[buf * KT + threadIdx.x] = bits >> threadIdx.x & 1 ? 0.f : NEG;
        return bits;
    };
    f32x16 acc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) acc[b] = splat16(0.f);
    ColumnScale<T, DB> cs;
    // p dp of 32 keys, dp less delta
    auto products = [&](int buf, int b, bool whole, f32x16& ds) {
        const T* kt = ks + buf * KT * KP;
        const T* vt = vs + buf * KT * VP;
        f32x16 st = whole ? splat16(0.f) : rows16(bias + buf * KT + 32 * b, lane);
        ds = splat16(-delta);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            st = Mma<T>::run(read_rows(kt, KP, 32 * b, 16 * s, lane), qf[s], st);
            ds = Mma<T>::run(read_rows(vt, VP, 32 * b, 16 * s, lane), of[s], ds);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) ds[j] *= __builtin_amdgcn_exp2f(fmaf(st[j], c, -lse2));
    };
    auto accumulate = [&](int buf, bool whole) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x16 ds[1];
            products(buf, b, whole, ds[0]);
            cs.apply(ds, acc);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> p = pack8<T>(ds[0], u);
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    acc[d] = Mma<T>::run(read_cols(ks + buf * KT * KP, KP, 32 * b + 16 * u, 32 * d, lane), p, acc[d]);
            }
        }
    };
    if (beg < end) fetch(beg);
    if constexpr (SHORT) {
        unsigned long long bits[2] = {0, 0};
#pragma unroll
        for (int t = 0; t < 2; ++t)
            if (t * KT < end) {
                bits[t] = stage(t * KT, t);
                if (t == 0 && KT < end) fetch(KT);
            }
        __syncthreads();
        float sum = 0.f;
        for (int t = 0; t * KT < end; ++t)
            if (bits[t]) {
                for (int b = 0; b < 2; ++b) {
                    f32x16 ds;
                    products(t, b, ~bits[t] == 0, ds);
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum += ds[j];
                }
            }
        delta = dfsfm::add_xor32(sum);
        if (r < R && lane < 32) a.delta[at] = delta;
        for (int t = 0; t * KT < end; ++t)
            if (bits[t]) accumulate(t, ~bits[t] == 0);
    } else {
        int buf = 0;
        for (int s0 = beg; s0 < end; s0 += KT, buf ^= 1) {
            const unsigned long long bits = stage(s0, buf);
            __syncthreads();
            if (s0 + KT < end) fetch(s0 + KT);
            if (bits) accumulate(buf, ~bits == 0);
        }
    }
    if (r >= R) return;
    const int64_t row = ((int64_t)job.n * a.L + l) * a.H + h;
    const float f = a.scale / cs.f;
    if (a.splits > 1)
        store_col<float, DB>(static_cast<float*>(a.o[0]) + job.split * a.numel + row * a.D, acc, f, a.D, lane);
    else
        store_col<T, DB>(static_cast<T*>(a.o[0]) + row * a.D, acc, f, a.D, lane);
}

// dk and dv: 4 waves x 32 keys a workgroup, tiles of 64 rows of q and dout, both read both ways.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dkdv_kernel(const Attn a) {
    constexpr int P = PITCH_T<T, DP>, DB = DP / 32, KS = DP / 16;
    // p of fp16 tensors times 2^14: a power of two that keeps weights down to 2^-28 exact and 1 in range
    constexpr float SHIFT = __is_same(T, f16) ? 14.f : 0.f, UNSHIFT = __is_same(T, f16) ? 1.f / 16384.f : 1.f;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* qs = reinterpret_cast<T*>(smem);
    T* os = qs + 2 * KT * P;
    float* rowv = reinterpret_cast<float*>(os + 2 * KT * P);              // [2][2][64]: -lse / scale, -delta
    const Job job(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hkv = a.H / a.G;
    const int s = job.tile * 128 + wave * 32 + (lane & 31);
    const int len = valid_len(a, job.n);
    bool there = s < len;
    if (a.mask) there = there && a.mask[(int64_t)job.n * a.S + min(s, a.S - 1)] != 0;
    // a tile is 64 queries of one of the G heads; splits take whole tiles
    const int lt = (a.L + KT - 1) / KT, per = (lt * a.G + a.splits - 1) / a.splits;
    const int beg = min(lt * a.G, job.split * per), end = min(lt * a.G, beg + per);

    Frag<T> kf[KS], vf[KS];
    const T* kp = static_cast<const T*>(a.k.p) + job.n * a.k.n + (int64_t)min(s, a.S - 1) * a.k.l + job.hk * a.k.h;
    const T* vp = static_cast<const T*>(a.v.p) + job.n * a.v.n + (int64_t)min(s, a.S - 1) * a.v.l + job.hk * a.v.h;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
        const int c = 16 * x + 8 * (lane >> 5);
        kf[x] = there && c < a.D ? load8<T>(kp + c) : zero_frag<T>();
        vf[x] = there && c < a.D ? load8<T>(vp + c) : zero_frag<T>();
    }
    const T* qb = static_cast<const T*>(a.q.p) + job.n * a.q.n + job.hk * a.G * a.q.h;
    const T* ob = static_cast<const T*>(a.dout.p) + job.n * a.dout.n + job.hk * a.G * a.dout.h;
    const int64_t vec = ((int64_t)job.n * a.H + job.hk * a.G) * a.L;
    Stage<T, DP> sq(a.q.l, a.D), so(a.dout.l, a.D);
    float rv = 0.f;                         // threads 0..63: -lse / scale of a row, 64..127: -delta
    int rows = 0;                           // rows of the tile in flight
    auto fetch = [&](int it) {
        const int g = it / lt, l0 = (it - g * lt) * KT;
        rows = a.L - l0;
        sq.load(qb + g * a.q.h + l0 * a.q.l, rows);
        so.load(ob + g * a.dout.h + l0 * a.dout.l, rows);
        if (threadIdx.x < 128) {
            const int row = threadIdx.x & 63;
            const int64_t at = vec + (int64_t)g * a.L + l0 + min(row, rows - 1);
            const float t = threadIdx.x < 64 ? a.lse[at] : a.delta[at];
            // a row without keys, or behind the last: a score of -inf, p = 0
            rv = threadIdx.x < 64 ? (row < rows && t != NEG ? -t / a.scale : NEG) : (row < rows ? -t : 0.f);
        }
    };
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) dk[b] = dv[b] = splat16(0.f);
    ColumnScale<T, DB> cs;
    const float c = a.scale * LOG2E;
    const bool any = __syncthreads_or(there);
    if (any && beg < end) fetch(beg);
    int buf = 0;
    for (int it = beg; any && it < end; ++it, buf ^= 1) {
        T* qt = qs + buf * KT * P;
        T* ot = os + buf * KT * P;
        float* vt = rowv + buf * 128;
        const unsigned long long keep = rows >= KT ? ~0ull : (1ull << rows) - 1;
        sq.store(qt, P, keep);
        so.store(ot, P, keep);
        if (threadIdx.x < 128) vt[threadIdx.x] = rv;
        __syncthreads();
        if (it + 1 < end) fetch(it + 1);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x16 st = rows16(vt + 32 * b, lane);
            f32x16 ds[1];
            ds[0] = rows16(vt + 64 + 32 * b, lane);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                st = Mma<T>::run(read_rows(qt, P, 32 * b, 16 * x, lane), kf[x], st);
                ds[0] = Mma<T>::run(read_rows(ot, P, 32 * b, 16 * x, lane), vf[x], ds[0]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                st[j] = __builtin_amdgcn_exp2f(fmaf(st[j], c, SHIFT));
                ds[0][j] *= st[j];
            }
            cs.apply(ds, dk);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> p = pack8<T>(st, u), g = pack8<T>(ds[0], u);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    dv[d] = Mma<T>::run(read_cols(ot, P, 32 * b + 16 * u, 32 * d, lane), p, dv[d]);
                    dk[d] = Mma<T>::run(read_cols(qt, P, 32 * b + 16 * u, 32 * d, lane), g, dk[d]);
                }
            }
        }
    }
    if (s >= a.S) return;
    if (!there) {                           // keys that are not there have no gradient, whatever q and dout hold
#pragma unroll
        for (int b = 0; b < DB; ++b) dk[b] = dv[b] = splat16(0.f);
    }
    const int64_t row = ((int64_t)job.n * a.S + s) * hkv + job.hk;
    const float f = a.scale * UNSHIFT / cs.f;
    if (a.splits > 1) {
        store_col<float, DB>(static_cast<float*>(a.o[0]) + job.split * a.numel + row * a.D, dk, f, a.D, lane);
        store_col<float, DB>(static_cast<float*>(a.o[1]) + job.split * a.numel + row * a.D, dv, UNSHIFT, a.D, lane);
    } else {
        store_col<T, DB>(static_cast<T*>(a.o[0]) + row * a.D, dk, f, a.D, lane);
        store_col<T, DB>(static_cast<T*>(a.o[1]) + row * a.D, dv, UNSHIFT, a.D, lane);
    }
}

// out = sum of the splits' partials, in their order
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* __restrict__ part, int64_t numel, int splits, T* __restrict__ out) {
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;      // D is a multiple of 8, so numel is
    if (e >= numel) return;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        float t[4];
        dfsfm::load_f32<float, 4>(part + s * numel + e, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += t[i];
    }
    dfsfm::store_f32<T, 4>(out + e, 4, o);
}

// ---------------------------------------------------------------- host
int pad_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// offsets within a tile of 64 rows are 32-bit byte offsets
bool stride_ok(int64_t l) { return l >= 0 && l < (1ll << 23); }

// Splits of the long axis (`length` rows of it, 256 a split at least).  512 workgroups run at a time (two a CU); as long as they number less
// than eight such rounds the last one's idle places count, and the smallest number of splits that fills 85 % of the places is taken: 608
// workgroups of the forward pass 2 x 4800 x 10816 x 8 x 32 fp32 take 1.21 ms, three splits of each 0.98 with the join.
int choose_splits(int64_t groups, int64_t length) {
    if (groups <= 0 || groups >= 4096) return 1;
    const int64_t most = length / 256 < 256 ? length / 256 : 256;
    int best = 1;
    double fill = 0;
    for (int s = 1; s <= most || s == 1; ++s) {
        const int64_t n = groups * s, places = (n + 511) / 512 * 512;
        const double f = (double)n / (double)places;
        if (f > fill + 0.02) fill = f, best = s;
        if (fill >= 0.85) break;
    }
    return best;
}

struct Plan {
    int heads, tq, tk, fwd, dq, dkdv;       // row tiles, key tiles, splits
    Plan(int N, int L, int S, int H, int Hkv) {
        heads = N * Hkv;
        const int64_t R = (int64_t)L * (H / Hkv);
        tq = (int)((R + 127) / 128);
        tk = (S + 127) / 128;
        fwd = dq = choose_splits((int64_t)heads * tq, S);
        dkdv = choose_splits((int64_t)heads * tk, R);
    }
};

bool shape_ok(int N, int L, int S, int H, int Hkv, int D) {
    if (D <= 0 || D > 128 || D % 8 || Hkv <= 0 || H % Hkv) return false;
    const int64_t R = (int64_t)L * (H / Hkv), heads = (int64_t)N * Hkv;
    // row and workgroup numbers are 32-bit
    return R < (1ll << 30) && S < (1 << 30) && heads < (1 << 20) && heads * ((R + 127) / 128 + 512) < (1ll << 31) &&
           heads * (((int64_t)S + 127) / 128 + 512) < (1ll << 31);
}

template <typename T, int DP>
int forward_dp(Attn a, const Plan& p, T* out, hipStream_t st) {
    constexpr int smem = 2 * KT * (PITCH<T, DP> + PITCH_T<T, DP>) * sizeof(T) + 2 * KT * 4;
    static dfsfm::SmemAttr attr;
    attr.ensure(reinterpret_cast<const void*>(&attn_forward_kernel<T, DP>), smem);
    a.tiles = p.tq;
    a.splits = p.fwd;
    if (p.fwd == 1) a.o[0] = out;
    hipLaunchKernelGGL((attn_forward_kernel<T, DP>), dim3((unsigned)(p.heads * p.tq * p.fwd)), dim3(256), smem, st, a);
    if (p.fwd > 1) {
        a.o[1] = out;
        const int64_t rows = (int64_t)a.N * a.L * a.H;
        hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, st, a);
    }
    return check_launch("dfsfm_cross_attention");
}

template <typename T, int DP>
int backward_dp(Attn a, const Plan& p, T* dq, T* dk, T* dv, float* part, hipStream_t st) {
    const int64_t rows = (int64_t)a.N * a.L * a.H, nq = rows * a.D, nk = (int64_t)a.N * a.S * (a.H / a.G) * a.D;
    if (rows > 0) {
        constexpr int smem = 2 * KT * (PITCH<T, DP> + PITCH_T<T, DP>) * sizeof(T) + 2 * KT * 4;
        const bool few = a.S <= 2 * KT;        // one split: choose_splits cuts from 256 keys up
        a.tiles = p.tq;
        a.splits = p.dq;
        a.numel = nq;
        a.o[0] = p.dq > 1 ? static_cast<void*>(part) : dq;
        const dim3 grid((unsigned)(p.heads * p.tq * p.dq));
        if (few) {
            static dfsfm::SmemAttr attr;
            attr.ensure(reinterpret_cast<const void*>(&attn_dq_kernel<T, DP, true>), smem);
            hipLaunchKernelGGL((attn_dq_kernel<T, DP, true>), grid, dim3(256), smem, st, a);
        } else {
            static dfsfm::SmemAttr attr;
            attr.ensure(reinterpret_cast<const void*>(&attn_dq_kernel<T, DP, false>), smem);
            hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, st, a);
            hipLaunchKernelGGL((attn_dq_kernel<T, DP, false>), grid, dim3(256), smem, st, a);
        }
        if (p.dq > 1)
            hipLaunchKernelGGL((attn_sum_kernel<T>), dim3((unsigned)((nq / 4 + 255) / 256)), dim3(256), 0, st, part, nq, p.dq, dq);
    }
    if (nk > 0) {
        constexpr int smem = 4 * KT * PITCH_T<T, DP> * sizeof(T) + 4 * KT * 4;
        static dfsfm::SmemAttr attr;
        attr.ensure(reinterpret_cast<const void*>(&attn_dkdv_kernel<T, DP>), smem);
        a.tiles = p.tk;
        a.splits = p.dkdv;
        a.numel = nk;
        a.o[0] = p.dkdv > 1 ? static_cast<void*>(part) : dk;
        a.o[1] = p.dkdv > 1 ? static_cast<void*>(part + p.dkdv * nk) : dv;
        hipLaunchKernelGGL((attn_dkdv_kernel<T, DP>), dim3((unsigned)(p.heads * p.tk * p.dkdv)), dim3(256), smem, st, a);
        if (p.dkdv > 1) {
            const dim3 grid((unsigned)((nk / 4 + 255) / 256));
            hipLaunchKernelGGL((attn_sum_kernel<T>), grid, dim3(256), 0, st, part, nk, p.dkdv, dk);
            hipLaunchKernelGGL((attn_sum_kernel<T>), grid, dim3(256), 0, st, part + p.dkdv * nk, nk, p.dkdv, dv);
        }
    }
    return check_launch("dfsfm_cross_attention_backward");
}

template <typename T>
int forward_any(const Attn& a, const Plan& p, void* out, hipStream_t st) {
    const int dp = pad_dim(a.D);
    return dp == 32 ? forward_dp<T, 32>(a, p, (T*)out, st) : dp == 64 ? forward_dp<T, 64>(a, p, (T*)out, st) : forward_dp<T, 128>(a, p, (T*)out, st);
}

template <typename T>
int backward_any(const Attn& a, const Plan& p, void* dq, void* dk, void* dv, float* part, hipStream_t st) {
    const int dp = pad_dim(a.D);
    return dp == 32   ? backward_dp<T, 32>(a, p, (T*)dq, (T*)dk, (T*)dv, part, st)
           : dp == 64 ? backward_dp<T, 64>(a, p, (T*)dq, (T*)dk, (T*)dv, part, st)
                      : backward_dp<T, 128>(a, p, (T*)dq, (T*)dk, (T*)dv, part, st);
}

}  // namespace

extern "C" size_t dfsfm_cross_attention_workspace(int N, int L, int S, int H, int Hkv, int D) {
    if (N <= 0 || L <= 0 || S < 0 || H <= 0 || !shape_ok(N, L, S, H, Hkv, D)) return 0;
    const Plan p(N, L, S, H, Hkv);
    return p.fwd > 1 ? (size_t)p.fwd * N * L * H * (D + 2) * sizeof(float) : 0;
}

extern "C" int dfsfm_cross_attention(const void* q, int64_t qn, int64_t ql, int64_t qh, const void* k, int64_t kn, int64_t ks, int64_t kh,
                                     const void* v, int64_t vn, int64_t vs, int64_t vh, const int* kv_lens, const uint8_t* kv_mask,
                                     void* out, float* lse, int N, int L, int S, int H, int Hkv, int D, float scale, int dtype,
                                     void* workspace, size_t workspace_bytes, void* stream_) {
    if (N == 0 || L == 0 || H == 0) return DFSFM_OK;
    if (!q || !out || !lse || (S > 0 && (!k || !v)) || N < 0 || L < 0 || S < 0 || H < 0 || !(scale > 0.f)) return DFSFM_E_BADARG;
    if (!shape_ok(N, L, S, H, Hkv, D)) return DFSFM_E_UNSUPPORTED;
    if (!stride_ok(ks) || !stride_ok(vs)) return DFSFM_E_UNSUPPORTED;
    if (workspace_bytes < dfsfm_cross_attention_workspace(N, L, S, H, Hkv, D)) return DFSFM_E_WORKSPACE;
    Attn a{};
    a.q = {q, qn, ql, qh};
    a.k = {k, kn, ks, kh};
    a.v = {v, vn, vs, vh};
    a.lens = kv_lens;
    a.mask = kv_mask;
    a.lse = lse;
    a.N = N, a.L = L, a.S = S, a.H = H, a.G = H / Hkv, a.D = D, a.scale = scale;
    a.numel = (int64_t)N * L * H * D;
    const Plan p(N, L, S, H, Hkv);
    a.o[0] = workspace;
    a.ml = static_cast<float*>(workspace) + p.fwd * a.numel;
    hipStream_t st = static_cast<hipStream_t>(stream_);
    if (dtype == DFSFM_F32) return forward_any<float>(a, p, out, st);
    if (dtype == DFSFM_BF16) return forward_any<bf16>(a, p, out, st);
    if (dtype == DFSFM_F16) return forward_any<f16>(a, p, out, st);
    return DFSFM_E_UNSUPPORTED;
}

extern "C" size_t dfsfm_cross_attention_backward_workspace(int N, int L, int S, int H, int Hkv, int D) {
    if (N <= 0 || L < 0 || S < 0 || H <= 0 || !shape_ok(N, L, S, H, Hkv, D)) return 0;
    const Plan p(N, L, S, H, Hkv);
    const size_t nq = (size_t)N * L * H, nk = (size_t)N * S * Hkv * D;
    const size_t a = p.dq > 1 ? p.dq * nq * D : 0, b = p.dkdv > 1 ? 2 * p.dkdv * nk : 0;
    return (nq + (a > b ? a : b)) * sizeof(float);
}

extern "C" int dfsfm_cross_attention_backward(const void* dout, int64_t gn, int64_t gl, int64_t gh, const void* q, int64_t qn, int64_t ql,
                                              int64_t qh, const void* k, int64_t kn, int64_t ks, int64_t kh, const void* v, int64_t vn,
                                              int64_t vs, int64_t vh, const void* out, int64_t on, int64_t ol, int64_t oh, const float* lse,
                                              const int* kv_lens, const uint8_t* kv_mask, void* dq, void* dk, void* dv, int N, int L, int S,
                                              int H, int Hkv, int D, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                              void* stream_) {
    if (N == 0 || H == 0 || (L == 0 && S == 0)) return DFSFM_OK;
    if (N < 0 || L < 0 || S < 0 || H < 0 || !(scale > 0.f)) return DFSFM_E_BADARG;
    if ((L > 0 && (!dout || !q || !out || !lse || !dq)) || (S > 0 && (!k || !v || !dk || !dv))) return DFSFM_E_BADARG;
    if (!shape_ok(N, L, S, H, Hkv, D)) return DFSFM_E_UNSUPPORTED;
    if (!stride_ok(ks) || !stride_ok(vs) || !stride_ok(ql) || !stride_ok(gl)) return DFSFM_E_UNSUPPORTED;
    if (workspace_bytes < dfsfm_cross_attention_backward_workspace(N, L, S, H, Hkv, D)) return DFSFM_E_WORKSPACE;
    Attn a{};
    a.q = {q, qn, ql, qh};
    a.k = {k, kn, ks, kh};
    a.v = {v, vn, vs, vh};
    a.dout = {dout, gn, gl, gh};
    a.out = {out, on, ol, oh};
    a.lens = kv_lens;
    a.mask = kv_mask;
    a.lse = const_cast<float*>(lse);
    a.N = N, a.L = L, a.S = S, a.H = H, a.G = H / Hkv, a.D = D, a.scale = scale;
    const Plan p(N, L, S, H, Hkv);
    a.delta = static_cast<float*>(workspace);
    float* part = a.delta + (int64_t)N * L * H;
    hipStream_t st = static_cast<hipStream_t>(stream_);
    if (dtype == DFSFM_F32) return backward_any<float>(a, p, dq, dk, dv, part, st);
    if (dtype == DFSFM_BF16) return backward_any<bf16>(a, p, dq, dk, dv, part, st);
    if (dtype == DFSFM_F16) return backward_any<f16>(a, p, dq, dk, dv, part, st);
    return DFSFM_E_UNSUPPORTED;
}
