// Softmax cross attention with its gradient -- gfx950 (MI355X).
//
//   forward   s = scale q k^T over the keys that are there, p = softmax(s), out = p v, lse = log sum exp(s); no key: out = 0, lse = -inf
//   backward  delta = <dout, out>, ds = p (dout v^T - delta), dq = scale ds k, dk = scale ds^T q, dv = p^T dout
//
// All products run on 32 x 32 MFMA tiles with 32-bit accumulators: bf16 and fp16 tensors on the 16-bit instruction, fp32 on it too, as three
// bf16 planes (X3), where many rows share a key, and on the 32-bit one where few do.  A lane holds ONE column of the score tile: a query in
// the forward and dq kernels, a key in the dk / dv kernel, so the running maximum, the sum and the scale of a query are per-lane values, and
// the accumulator registers of a score tile are, in their order, the operand of the next product (its other operand is read from LDS with the
// same order of the inner index): the scores never leave the registers.  The query heads that share a key head are rows of one problem: row
// r is (query r / G, head r % G).
//
// Tiles come by LDS-DMA, the next one while this one is worked on, save where waiting for it is faster (Few, attn_dkdv_kernel).  Keys behind
// kv_lens are out of the DMA descriptor's range and arrive as zeros; rows of LDS whose kv_mask is 0 are cleared; scores of both are set to
// -inf; a tile without any key is skipped.  Few rows: the keys (or, for dk / dv, the rows) are cut into splits that write 32-bit partial
// results, joined in a fixed order by a second kernel.  No atomics.
//
// What bounds the large cases is the exponentials beside the products: a wave's VALU instructions run at half rate while the other wave of its
// SIMD streams MFMAs.  4 x 4800 x 6400 keys (ragged) x 16 / 4 heads x 128 bf16: forward 0.69 - 0.74, dq 0.85 - 0.89, dk / dv 1.10 - 1.19 ms by
// the card, in products 0.83 - 0.89, 1.04 - 1.09 and 1.04 - 1.12 PFLOP/s, where a plain 8192^3 product of the library runs at 1.17; the
// matrix pipes are busy 41, 55 and 52 % of the time.  fp32, 2 x 4800 x 4800 x 8 heads: forward at D = 32 295 us = 160 TFLOP/s, 64 495 = 190,
// 128 1100 = 172 (library: 154), with the gradient 1.18, 2.13 and 4.67 ms = 140, 154 and 141; D = 40, 80 and 96 pay for 64, 128 and 128
// (0.45, 1.03 and 1.04 ms forward): blocks of channels that are not there are multiplied, since the chunk order in LDS takes powers of two.
#include "elem.h"

namespace {

using dfsfm::bf16;
using dfsfm::f16;
using dfsfm::check_launch;
using dfsfm::mfma32_row;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
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

// fp32 as three bf16 planes: 24 bits of mantissa are 8 + 8 + 8, so x = a + b + c exactly (down to 2^-126), with fp32's range.  A product is
// six 16-bit matrix instructions, the terms above 2^-24 of it, in 192 cycles where eight 32-bit ones take 512.
struct X3;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct Frag3 {
    bf16x8 p[3];
};
template <>
struct Mma<X3> {
    typedef Frag3 frag;
    static __device__ __forceinline__ f32x16 run(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
        for (int i = 2; i >= 0; --i)                                      // small terms first
#pragma unroll
            for (int j = i; j >= 0; --j) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[i - j], b.p[j], c, 0, 0, 0);
        return c;
    }
};

template <typename T>
using Frag = typename Mma<T>::frag;

// What tensors hold in memory, what tiles hold in LDS, planes of a tile.
template <typename T>
struct Type {
    typedef T mem, elem;
    static constexpr int PLANES = 1;
};
template <>
struct Type<X3> {
    typedef float mem;
    typedef bf16 elem;
    static constexpr int PLANES = 3;
};
template <typename T>
using Mem = typename Type<T>::mem;
template <typename T>
using Elem = typename Type<T>::elem;

// The planes of 8 values.  FINITE values only: infinity less infinity is no rest.
template <bool FINITE>
__device__ __forceinline__ Frag3 split8(const float (&x)[8]) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    Frag3 f;
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(__float_as_uint(r[2 * j + 1]), __float_as_uint(r[2 * j]), 0x07060302);
        f.p[k] = __builtin_bit_cast(bf16x8, w);
        if (k < 2)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float rest = r[j] - __uint_as_float(__float_as_uint(r[j]) & 0xffff0000u);
                r[j] = FINITE || fabsf(x[j]) != INFINITY ? rest : 0.f;
            }
    }
    return f;
}

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
    if constexpr (__is_same(T, X3)) {
        const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        return split8<true>(z);
    } else {
        Frag<T> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (T)0.f;
        return f;
    }
}

// 8 consecutive channels from global memory
template <typename T>
__device__ __forceinline__ Frag<T> load8(const Mem<T>* p) {
    if constexpr (__is_same(T, X3)) {
        typedef f32x8 at16 __attribute__((aligned(16)));
        const f32x8 v = *reinterpret_cast<const at16*>(p);
        const float x[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        return split8<false>(x);
    } else {
        typedef Frag<T> at16 __attribute__((aligned(16)));
        return *reinterpret_cast<const at16*>(p);
    }
}

// How a tile of DP channels a row lies in LDS, and where this lane reads it.  Both ways of reading have to spread over all 64 banks: as A
// operands (16 bytes a lane, a row a lane) and transposed (16 lanes read four rows x 32 bytes).  Rows have no padding (the tile is written
// by LDS-DMA, 1 KB of consecutive LDS an instruction); their 16-byte chunks are permuted by the row number: chunk c of row r lies at c ^
// order(r), where order() differs by at least four chunks between neighbouring rows that share banks (the transposed read) and takes every
// value over 16 rows (the other).  A lane's row is the same modulo 16 in every read, so the permutation is one exclusive or with a
// constant.  Padded rows (272 or 288 bytes) cost the dk / dv kernel 35 % of its LDS cycles in conflicts; this order has none, by the counter in
// every kernel of this file.
template <typename T, int DP>
struct LdsPlane {
    static constexpr bool HALF = sizeof(T) == 2;
    static constexpr int CH = DP * sizeof(T) / 16, E = 16 / sizeof(T);    // chunks a row, elements a chunk
    int rows, cols;                                                       // this lane's offsets
    static __host__ __device__ constexpr int order(int r) {
        return CH >= 16 ? (r & 3) << 2 | (r >> 2 & 3) : CH == 8 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : r >> 2 & 3;
    }
    __device__ __forceinline__ explicit LdsPlane(int lane) {
        const int i = lane & 15, half = lane >> 5, r = 4 * half + (i >> 2);
        rows = (lane & 31) * DP + ((HALF ? half : 2 * half) ^ order(lane & 31)) * E;
        cols = HALF ? r * DP + (((lane & 16) / 8 + (i >> 1 & 1)) ^ order(r)) * E + 4 * (i & 1) : 4 * half * DP + ((lane & 31) ^ order(4 * half) * E);
    }
    // A operand: rows row .. row + 31 (row: a multiple of 32), inner index = channels col .. col + 15
    __device__ __forceinline__ Frag<T> read_rows(const T* tile, int row, int col) const {
        const T* p = tile + row * DP;
        if constexpr (HALF) {
            return *reinterpret_cast<const Frag<T>*>(p + (rows ^ col));
        } else {
            const f32x4 u = *reinterpret_cast<const f32x4*>(p + (rows ^ col)), v = *reinterpret_cast<const f32x4*>(p + (rows ^ col ^ E));
            return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // A operand of the transposed tile: rows = channels col .. col + 31, inner index = tile rows row .. row + 15 in the order of an
    // accumulator's registers: slot j of half h is row + (j & 3) + 8 (j >> 2) + 4 h
    __device__ __forceinline__ Frag<T> read_cols(const T* tile, int row, int col) const {
        const T* p = tile + row * DP;
        if constexpr (HALF) {
            // 16 lanes read a 4 x 16 block, 8 bytes each along its rows; the transposed read hands lane i the block's column i
            typedef __attribute__((address_space(3))) s16x4* lds_ptr;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + (cols ^ col)));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * DP + (cols ^ col ^ order(8) * E)));
            return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            Frag<T> f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = p[((j & 3) + 8 * (j >> 2)) * DP + (cols ^ col ^ order((j & 3) + 8 * (j >> 2)) * E)];
            return f;
        }
    }
};

// Rows of a staged tile: 64, 32 where three planes of 64 channels or more would leave one workgroup a CU.
template <typename T, int DP>
constexpr int ROWS = __is_same(T, X3) && DP >= 64 ? 32 : 64;

// The planes of a tile, one behind the other.
template <typename T, int DP>
struct Lds : LdsPlane<Elem<T>, DP> {
    typedef LdsPlane<Elem<T>, DP> Plane;
    static constexpr int PLANES = Type<T>::PLANES, PLANE = ROWS<T, DP> * DP, TILE = PLANES * PLANE;
    using Plane::Plane;
    __device__ __forceinline__ Frag<T> read_rows(const Elem<T>* tile, int row, int col) const {
        if constexpr (PLANES == 1) {
            return Plane::read_rows(tile, row, col);
        } else {
            return {Plane::read_rows(tile, row, col), Plane::read_rows(tile + PLANE, row, col), Plane::read_rows(tile + 2 * PLANE, row, col)};
        }
    }
    __device__ __forceinline__ Frag<T> read_cols(const Elem<T>* tile, int row, int col) const {
        if constexpr (PLANES == 1) {
            return Plane::read_cols(tile, row, col);
        } else {
            return {Plane::read_cols(tile, row, col), Plane::read_cols(tile + PLANE, row, col), Plane::read_cols(tile + 2 * PLANE, row, col)};
        }
    }
};

// Registers 8 t .. 8 t + 7 of a score tile as the other operand (round to nearest even).
template <typename T>
__device__ __forceinline__ Frag<T> pack8(const f32x16& s, int t) {
    if constexpr (__is_same(T, X3)) {
        const float x[8] = {s[8 * t], s[8 * t + 1], s[8 * t + 2], s[8 * t + 3], s[8 * t + 4], s[8 * t + 5], s[8 * t + 6], s[8 * t + 7]};
        return split8<true>(x);
    } else {
        Frag<T> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (T)s[8 * t + j];
        return f;
    }
}
// FINE kernels: 8 values as the sum of two operands.  16-bit weights (or gradients) are off by as much as a 16-bit result is, and a result of
// rounded ones by sqrt(2) of that, which many results share out evenly and few do not.  Where few rows read their keys once, from memory, a
// second product takes 0 - 8 % more time, and only the result's own rounding is left (single tokens x 10816 keys fp16: 3.0e-4 -> 2.1e-4 off in the 2-norm).
// 7/8 of the value and the rest: the error is that of 1/8 of it, and both have its sign, so that an infinite factor stays what it is.
template <typename T>
struct Fine {
    Frag<T> p, rest;
    __device__ __forceinline__ Fine(const f32x16& s, int t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (T)(0.875f * s[8 * t + j]);
        asm("" : "+v"(p));                  // one p: the compiler may round a tie once for the product and otherwise, fused, for the rest
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = (T)(s[8 * t + j] - (float)p[j]);
    }
    // acc + x s
    __device__ __forceinline__ f32x16 times(const Frag<T>& x, const f32x16& acc) const { return Mma<T>::run(x, rest, Mma<T>::run(x, p, acc)); }
};
template <typename T>
struct Packed {
    Frag<T> p;
    __device__ __forceinline__ Packed(const f32x16& s, int t) : p(pack8<T>(s, t)) {}
    __device__ __forceinline__ f32x16 times(const Frag<T>& x, const f32x16& acc) const { return Mma<T>::run(x, p, acc); }
};
template <typename T, bool FINE>
struct OperandOf { typedef Packed<T> type; };
template <typename T>
struct OperandOf<T, true> { typedef Fine<T> type; };
template <typename T, bool FINE>
using Operand = typename OperandOf<T, FINE>::type;

// Waves a SIMD that the forward and dq kernels are compiled for: two (256 registers a wave), so that one wave's exponentials run beside the
// other's products.  fp32 at D = 128 holds twice the operands and would spill.
template <typename T, int DP>
constexpr int WAVES = sizeof(Mem<T>) == 4 && DP == 128 ? 1 : 2;

struct Tensor {
    const void* p;
    int64_t n, l, h;                       // element strides of [N, length, heads, D]; the channel stride is 1
};

struct Attn {
    Tensor q, k, v, dout, out;
    Tensor qt, kt, vt, dt;                 // q, k, v, dout as tiles are fetched from: themselves, or the first of their planes
    int64_t plane_q, plane_k;              // elements between planes
    const int* lens;
    const uint8_t* mask;                   // [N, S]
    void* o[2];                            // results (out, or dq, or dk and dv): dense, in T or, with splits, 32-bit partials
    float* lse;                            // [N, H, L]
    f32x4* ml;                             // forward partials: reference, sum, sum of rounded weights [splits][N, H, L]
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
    __device__ __forceinline__ Job(const Attn& a, int tiles, int splits) {
        const int hkv = a.H / a.G, heads = a.N * hkv;
        tile = blockIdx.x % tiles;
        const int rest = blockIdx.x / tiles, head = rest % heads;
        split = rest / heads;
        n = head / hkv;
        hk = head % hkv;
    }
    __device__ __forceinline__ explicit Job(const Attn& a) : Job(a, a.tiles, a.splits) {}
    // The same for tiles of `rows` keys, the tiles with keys of every sequence first: workgroups go to XCDs by their number, so tiles that
    // have nothing to do must not lie between the others (4 x 6400 ragged keys: XCDs with four rounds of work beside ones with three).
    // Every workgroup walks the lengths, which more sequences do not repay: 256 single tokens x 2048 x 8 x 64 take 131 us as they come, 210
    // sorted, 128 x 512 x 512 forward and gradient 384 and 422; 64 x 512 x 512 206 and 212, 4 x 4800 x 6400 (see above) gains.
    __device__ __forceinline__ Job(const Attn& a, int tiles, int splits, int rows) : Job(a, tiles, splits) {
        if (!a.lens || a.N > 64) return;
        const int hkv = a.H / a.G, per = hkv * splits;
        unsigned id = blockIdx.x;
        for (int pass = 0; pass < 2; ++pass)
            for (int i = 0; i < a.N; ++i) {
                const int with = (min(max(a.lens[i], 0), a.S) + rows - 1) / rows, count = pass ? tiles - with : with;
                if (id < (unsigned)(count * per)) {
                    n = i;
                    tile = (pass ? with : 0) + id % count;
                    hk = id / count % hkv;
                    split = id / count / hkv;
                    return;
                }
                id -= count * per;
            }
    }
};

__device__ __forceinline__ int valid_len(const Attn& a, int n) { return a.lens ? min(max(a.lens[n], 0), a.S) : a.S; }

// A tile of NROWS rows x DP channels on its way from memory into LDS, by LDS-DMA: no register holds it and no vector instruction moves it.
// Every one of THREADS threads (the workgroup, or a wave for itself) fetches 16 bytes an instruction; the chunk order of Lds is applied to the
// source address.  Rows behind the last and channels behind D lie outside the buffer descriptor and arrive as zeros.
template <typename T, int DP, int NROWS, int THREADS>
struct Dma {
    typedef LdsPlane<Elem<T>, DP> L;
    static constexpr int CH = L::CH, PER = NROWS * CH / THREADS, RPI = THREADS / CH;   // instructions a plane, rows an instruction
    static_assert(NROWS * CH % THREADS == 0, "every thread fetches the same number of chunks");
    int64_t plane;
    unsigned tid, off, step, row_bytes, stride;
    __device__ __forceinline__ Dma(int64_t stride_, int D, int64_t plane_) : plane(plane_), stride((unsigned)(stride_ * sizeof(Elem<T>))) {
        row_bytes = D * (unsigned)sizeof(Elem<T>);
        tid = threadIdx.x % THREADS;
        off = tid / CH * stride;
        step = RPI * stride;
    }
    // rows base .. base + rows - 1 (rows > 0); base, rows and tile are the same in every lane
    __device__ __forceinline__ void issue(const Elem<T>* base, int rows, Elem<T>* tile) const {
#pragma unroll
        for (int k = 0; k < Type<T>::PLANES; ++k) issue_plane(base + k * plane, rows, tile + k * NROWS * DP);
    }
    __device__ __forceinline__ void issue_plane(const Elem<T>* base, int rows, Elem<T>* tile) const {
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint64_t at = reinterpret_cast<uint64_t>(base);
        const i32x4 rsrc = {__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                            __builtin_amdgcn_readfirstlane((int)((unsigned)(min(rows, NROWS) - 1) * stride + row_bytes)), 0x00020000};
        const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)tile) + wave * 1024;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned c = (tid % CH ^ L::order(tid / CH) ^ L::order(RPI * i & 15)) * 16;
            // channels behind D: an offset no descriptor reaches (strides are below 2^23 elements)
            const unsigned o = c < row_bytes ? off + step * i + c : 0xff000000u;
            // As assembly (it writes no register) because the compiler lets every LDS read wait for its own form of this load.  The waits:
            // five states from a lane read's scalar to a memory instruction that uses it, one from m0 (which nothing else here uses).
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to + i * THREADS * 16), "v"(o), "s"(rsrc) : "memory");
        }
    }
};

__device__ __forceinline__ void dma_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Operands that a loop of tiles reads again and again have to be in their registers before it: the compiler knows of their loads but not of
// the tiles'.  A load that is not settled for it, it waits for in the loop, before the product, until every load is done, the next tile's
// among them (tests/test_train_edges_cpu.py looks for such waits in the assembly).
template <typename T, int N>
__device__ __forceinline__ void settle(Frag<T> (&f)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) {
        if constexpr (__is_same(T, X3)) {
#pragma unroll
            for (int k = 0; k < 3; ++k) asm volatile("" : "+v"(f[s].p[k]));
        } else {
            asm volatile("" : "+v"(f[s]));
        }
    }
}

// Zeros over the rows of a tile whose bit in `keep` is 0, by 256 threads.
template <typename T, int DP>
__device__ __forceinline__ void zero_rows(Elem<T>* tile, unsigned long long keep) {
    typedef Lds<T, DP> L;
    unsigned e = threadIdx.x;
    asm volatile("" : "+v"(e));            // keeps this branch's addresses out of the loop's registers
#pragma unroll
    for (int i = 0; i < L::TILE / L::E / 256; ++i, e += 256)
        if (!(keep >> (e / L::CH % ROWS<T, DP>) & 1)) *reinterpret_cast<f32x4*>(tile + e * L::E) = f32x4{0.f, 0.f, 0.f, 0.f};
}

// The mask byte of key s0 + lane, one tile ahead of its use; 1 without a mask.
__device__ __forceinline__ unsigned key_mask(const Attn& a, int n, int s0) {
    return a.mask ? a.mask[(int64_t)n * a.S + min(s0 + (int)(threadIdx.x & 63), a.S - 1)] : 1u;
}

// Bits of the KT keys from s0 on that are there; the same in every wave.
template <int KT>
__device__ __forceinline__ unsigned long long key_bits(unsigned mask, int s0, int end) {
    const int i = threadIdx.x & 63;
    return __ballot(i < KT && s0 + i < end && mask != 0);
}
template <int KT>
constexpr unsigned long long ALL_KEYS = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;

// Scores of keys that are not there become -inf, whatever they were: bits of 32 keys, this lane's half shifted to bit 0.
__device__ __forceinline__ void drop_keys(f32x16& st, unsigned bits) {
#pragma unroll
    for (int j = 0; j < 16; ++j) st[j] = bits >> mfma32_row(j, 0) & 1 ? st[j] : NEG;
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

// sum + the 8 weights of an operand, as they were rounded.  out is divided by this sum and not by that of the weights before rounding: it
// stays a mean of values of v (v at fp16's largest value gives that value, not infinity; a row that one key dominates is exact), while lse
// keeps the 32-bit sum.  One instruction for two weights.
template <typename T>
__device__ __forceinline__ float add_rounded(const Frag<T>& f, float sum) {
    if constexpr (__is_same(T, bf16)) {
        typedef bf16 v2 __attribute__((ext_vector_type(2)));
        const v2 one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_fdot2_f32_bf16(v2{f[2 * j], f[2 * j + 1]}, one, sum, false);
    } else if constexpr (__is_same(T, f16)) {
        typedef f16 v2 __attribute__((ext_vector_type(2)));
        const v2 one = {(f16)1.f, (f16)1.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_fdot2(v2{f[2 * j], f[2 * j + 1]}, one, sum, false);
    }
    return sum;
}
// whether a type's weights are rounded before their product
template <typename T>
constexpr bool ROUNDS = !__is_same(T, float) && !__is_same(T, X3);

// Stores a transposed accumulator (channels x columns) to the dense row of this lane's column.  A lane holds 4 of every 8 channels; in 16
// bits its partner's 4 are swapped in for every second eight, so that each stores 16 bytes: half the write requests of 8-byte stores.
template <typename T, int DB>
__device__ __forceinline__ void store_col(T* row, const f32x16 (&acc)[DB], float f, int D, int lane) {
#pragma unroll
    for (int b = 0; b < DB; ++b) {
        if constexpr (sizeof(T) == 2) {
            typedef T v4 __attribute__((ext_vector_type(4)));
            typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
            typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                v4 x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = (T)(acc[b][4 * g + e] * f);
                    y[e] = (T)(acc[b][4 * g + 4 + e] * f);
                }
                const u32x2 u = __builtin_bit_cast(u32x2, x), v = __builtin_bit_cast(u32x2, y);
                // lower half: its own and its partner's eight g; upper half: eight g + 1
                const auto p = __builtin_amdgcn_permlane32_swap(u[0], v[0], false, false), q = __builtin_amdgcn_permlane32_swap(u[1], v[1], false, false);
                const int d = 32 * b + 8 * g + 8 * (lane >> 5);
                if (d < D) *reinterpret_cast<u32x4*>(row + d) = u32x4{p[0], q[0], p[1], q[1]};         // D is a multiple of 8
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * b + 8 * g + 4 * (lane >> 5);
                if (d < D) *reinterpret_cast<f32x4*>(row + d) = f32x4{acc[b][4 * g] * f, acc[b][4 * g + 1] * f, acc[b][4 * g + 2] * f, acc[b][4 * g + 3] * f};
            }
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
        if constexpr (__is_same(T, f16)) {
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
__device__ __forceinline__ float inverse(float sum) { return sum > 0.f || sum != sum ? 1.f / sum : 0.f; }
// log sum exp of a row from its reference (in powers of two) and its sum; -inf without keys
__device__ __forceinline__ float log_sum(float m, float sum) { return fmaf(m == NEG ? 0.f : m, LN2, logf(sum)); }

// A wave's 32 columns of queries on their way through the keys.
//
// The reference m lies LIFT powers of two under the largest score it was taken from and follows once scores are 8 further above it.  fp16
// weights then reach 2^15 and a row's largest is 2^7 or above: what rounds to a subnormal, by up to 2^-25, is off by 2^-32 of the largest.
// With the reference at the largest score, weights under 2^-25 of it were 0: behind a first key that holds a row's weight, 9000 keys e^-17.5
// below it came out up to a fifth off.
template <typename T, int DP, int KT = ROWS<T, DP>, bool FINE = false>
struct Softmax {
    static constexpr int DB = DP / 32, KS = DP / 16;
    static constexpr float LIFT = __is_same(T, f16) ? 7.f : 0.f;
    f32x16 acc[DB];
    float m = NEG, sum = 0.f, rsum = 0.f;   // reference in powers of two of scale * log2(e) * q k; sums of this lane's half of the keys
    const float c;
    __device__ __forceinline__ explicit Softmax(float scale) : c(scale * LOG2E) {
#pragma unroll
        for (int b = 0; b < DB; ++b) acc[b] = splat16(0.f);
    }
    // A tile's second half without keys (a short sequence's last tile) is left out: 4800 x 77 x 64 29 -> 26 us.  At D = 128 the second copy of
    // the code costs the loop its registers.
    __device__ __forceinline__ void tile(const Lds<T, DP>& lds, const Elem<T>* kt, const Elem<T>* vt, const Frag<T> (&qf)[KS], unsigned long long bits, int lane) {
        if (KT == 64 && DP < 128 && bits >> 32 == 0)
            blocks<1>(lds, kt, vt, qf, bits, lane);
        else
            blocks<KT / 32>(lds, kt, vt, qf, bits, lane);
    }
    template <int NB>
    __device__ __forceinline__ void blocks(const Lds<T, DP>& lds, const Elem<T>* kt, const Elem<T>* vt, const Frag<T> (&qf)[KS], unsigned long long bits, int lane) {
        f32x16 st[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            st[b] = splat16(0.f);
#pragma unroll
            for (int s = 0; s < KS; ++s) st[b] = Mma<T>::run(lds.read_rows(kt, 32 * b, 16 * s), qf[s], st[b]);
        }
        if (bits != ALL_KEYS<KT>) {
#pragma unroll
            for (int b = 0; b < NB; ++b) drop_keys(st[b], (unsigned)(bits >> 32 * b >> 4 * (lane >> 5)));
        }
        float t = NEG;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) t = fmaxf(t, st[b][j]);
        t = fmaxf(t, dfsfm::from_xor32(t, lane)) * c;
        // the reference follows the maximum once it is 8 behind: weights up to 2^8 lose nothing, and most tiles rescale nothing
        if (__ballot(t > m + (8.f + LIFT))) {
            const float mn = t > m + (8.f + LIFT) ? t - LIFT : m, f = m == NEG ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            sum *= f;
            rsum *= f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[b][j] *= f;
        }
        const float mm = m == NEG ? 0.f : m;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                st[b][j] = __builtin_amdgcn_exp2f(fmaf(st[b][j], c, -mm));
                sum += st[b][j];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Operand<T, FINE> p(st[b], u);
                if constexpr (!FINE) rsum = add_rounded<T>(p.p, rsum);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = p.times(lds.read_cols(vt, 32 * b + 16 * u, 32 * d), acc[d]);
            }
        }
    }
    __device__ __forceinline__ void finish() {
        sum = dfsfm::add_xor32(sum);
        rsum = ROUNDS<T> && !FINE ? dfsfm::add_xor32(rsum) : sum;
    }
};

// 4 waves x 32 rows a workgroup; tiles of 64 keys, two in LDS.
template <typename T, int DP>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void attn_forward_kernel(const Attn a) {
    constexpr int DB = DP / 32, KS = DP / 16, TILE = Lds<T, DP>::TILE, KT = ROWS<T, DP>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Elem<T>* ks = reinterpret_cast<Elem<T>*>(smem);
    Elem<T>* vs = ks + 2 * TILE;
    const Job job(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Lds<T, DP> lds(lane);
    const int R = a.L * a.G, r = job.tile * 128 + wave * 32 + (lane & 31);
    const int l = r / a.G, h = job.hk * a.G + r % a.G;
    const int len = valid_len(a, job.n);
    const int per = ((len + KT - 1) / KT + a.splits - 1) / a.splits * KT;   // keys a split, whole tiles
    const int beg = min(len, job.split * per), end = min(len, beg + per);

    Frag<T> qf[KS];
    const Mem<T>* qp = static_cast<const Mem<T>*>(a.q.p) + job.n * a.q.n + (int64_t)min(l, a.L - 1) * a.q.l + h * a.q.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * (lane >> 5);
        qf[s] = r < R && c < a.D ? load8<T>(qp + c) : zero_frag<T>();
    }
    const Elem<T>* kb = static_cast<const Elem<T>*>(a.kt.p) + job.n * a.kt.n + job.hk * a.kt.h;
    const Elem<T>* vb = static_cast<const Elem<T>*>(a.vt.p) + job.n * a.vt.n + job.hk * a.vt.h;
    const Dma<T, DP, KT, 256> dk(a.kt.l, a.D, a.plane_k), dv(a.vt.l, a.D, a.plane_k);
    unsigned mask = 0;
    auto fetch = [&](int s0, int buf) {
        dk.issue(kb + s0 * a.kt.l, end - s0, ks + buf * TILE);
        dv.issue(vb + s0 * a.vt.l, end - s0, vs + buf * TILE);
        mask = key_mask(a, job.n, s0);
    };
    Softmax<T, DP> sm(a.scale);
    const bool mine = job.tile * 128 + wave * 32 < R;
    if (beg < end) fetch(beg, 0);
    int buf = 0;
    for (int s0 = beg; s0 < end; s0 += KT, buf ^= 1) {
        const Elem<T>* kt = ks + buf * TILE;
        Elem<T>* vt = vs + buf * TILE;
        dma_landed();
        const unsigned long long bits = key_bits<KT>(mask, s0, end);
        __syncthreads();                    // all of the tile is there, and the other buffer's readers are done
        if (a.mask && bits != ALL_KEYS<KT> && bits) {      // a weight of 0 does not undo a NaN in v
            zero_rows<T, DP>(vt, bits);
            __syncthreads();
        }
        if (s0 + KT < end) fetch(s0 + KT, buf ^ 1);
        if (bits != 0 && mine) sm.tile(lds, kt, vt, qf, bits, lane);
    }
    sm.finish();
    if (r >= R) return;
    const int64_t row = ((int64_t)job.n * a.L + l) * a.H + h, at = ((int64_t)job.n * a.H + h) * a.L + l;
    if (a.splits > 1) {
        store_col<float, DB>(static_cast<float*>(a.o[0]) + job.split * a.numel + row * a.D, sm.acc, 1.f, a.D, lane);
        if (lane < 32) a.ml[(int64_t)job.split * a.N * a.H * a.L + at] = f32x4{sm.m, sm.sum, sm.rsum, 0.f};
    } else {
        store_col<Mem<T>, DB>(static_cast<Mem<T>*>(a.o[0]) + row * a.D, sm.acc, inverse(sm.rsum), a.D, lane);
        if (lane < 32) a.lse[at] = log_sum(sm.m, sm.sum);
    }
}

// Up to 32 rows a head, the single-token form: bound by the keys' bytes.  Every wave walks its own tiles of 32 keys through its own ring in
// LDS, without a barrier; the waves' results meet in LDS at the end.  A workgroup's rings are 64 KB (16 a wave), two workgroups a CU, where
// that holds two stages or more (16 bits up to 64 channels, fp32 up to 32), and 128 KB, one a CU, for wider rows.  With a mask a turn waits for
// every tile in flight: its byte is loaded where it is used, and the compiler's wait for it counts no tiles.  32 single tokens x 8192 keys x
// 8 x 64 fp16: 98 us, 5.5 TB/s; 16 x 10816 ragged keys: 52 - 59 us with the join, 3.4 - 3.9 TB/s (the kernel above, whose four waves share
// each tile: 117 and 60), 81 with a mask of two thirds.
template <typename T, int DP>
struct Few {
    static constexpr int KT = 32, TILE = KT * DP, STAGE = 2 * TILE * sizeof(T);       // K and V
    static constexpr int WAVES = STAGE > 16384 ? 2 : 4, STAGES = STAGE > 8192 ? 2 : 16384 / STAGE, PITCH = DP + 4;
    static constexpr int RING = WAVES * STAGES * STAGE, JOIN = WAVES * 32 * (PITCH + 4) * 4;
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
    // Where two workgroups of two stages share a CU, q is left unsettled: the compiler's wait then takes the next tile in, between the reads of
    // this one and their products.  32 tokens x 8192 x 8 x 64 fp16 take 98 us so, 104 with the products beside the next tile's fetch, 16 x
    // 4096 x 8 x 32 fp32 37 and 38.  With more stages, or one workgroup, it is the other way: 32 x 8192 x 8 x 32 bf16 84 and 82, x 128 fp16
    // 181 and 178, 16 x 8192 x 8 x 64 fp32 132 and 116.
    static constexpr bool NEXT_TOO = STAGES == 2 && RING == 65536;
};
template <typename T, int DP>
__global__ __launch_bounds__((64 * Few<T, DP>::WAVES)) void attn_forward_few_kernel(const Attn a) {
    typedef Few<T, DP> F;
    constexpr int DB = DP / 32, KS = DP / 16, KT = F::KT, TILE = F::TILE, NW = F::WAVES, NS = F::STAGES;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // splits are as long in every sequence, so that those that are there take as long
    const int per = ((a.S + KT * NW - 1) / (KT * NW) + a.splits - 1) / a.splits * KT * NW;
    const Job job(a, a.splits, 1, max(per, 1));
    const int split = job.tile;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    T* ring = reinterpret_cast<T*>(smem) + wave * NS * 2 * TILE;
    const Lds<T, DP> lds(lane);
    const int R = a.L * a.G, r = lane & 31, l = r / a.G, h = job.hk * a.G + r % a.G;
    const int len = valid_len(a, job.n);
    const int end = (int)min((int64_t)len, (int64_t)(split + 1) * per), beg = min(end, (int)min((int64_t)end, (int64_t)split * per) + wave * KT);
    Frag<T> qf[KS];
    const T* qp = static_cast<const T*>(a.q.p) + job.n * a.q.n + (int64_t)min(l, a.L - 1) * a.q.l + h * a.q.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * (lane >> 5);
        qf[s] = r < R && c < a.D ? load8<T>(qp + c) : zero_frag<T>();
    }
    const T* kb = static_cast<const T*>(a.k.p) + job.n * a.k.n + job.hk * a.k.h;
    const T* vb = static_cast<const T*>(a.v.p) + job.n * a.v.n + job.hk * a.v.h;
    const Dma<T, DP, KT, 64> dk(a.k.l, a.D, 0), dv(a.v.l, a.D, 0);
    constexpr int LOADS = dk.PER + dv.PER;
    auto fetch = [&](int s0, int stage) {
        T* at = ring + stage * 2 * TILE;
        dk.issue(kb + s0 * a.k.l, end - s0, at);
        dv.issue(vb + s0 * a.v.l, end - s0, at + TILE);
    };
    Softmax<T, DP, KT, ROUNDS<T>> sm(a.scale);
    if constexpr (F::NEXT_TOO) dma_landed();
    else settle<T>(qf);                     // q is here: from now on the counter counts tiles
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
        if (beg + i * KT * NW < end) fetch(beg + i * KT * NW, i);
    int stage = 0;
    for (int s0 = beg; s0 < end; s0 += KT * NW) {
        // the stage after the last in flight was read in the turn before; its reads are done, their results went into products
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int ahead = s0 + (NS - 1) * KT * NW;
        if (ahead < end) {
            fetch(ahead, stage ? stage - 1 : NS - 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * LOADS) : "memory");
        } else {
            dma_landed();
        }
        T* at = ring + stage * 2 * TILE;
        const unsigned long long bits = key_bits<KT>(key_mask(a, job.n, s0), s0, end);
        if (a.mask && bits != ALL_KEYS<KT>) {                 // a weight of 0 does not undo a NaN in v
            for (int e = lane; e < TILE / lds.E; e += 64)
                if (!(bits >> (e / lds.CH) & 1)) *reinterpret_cast<f32x4*>(at + TILE + e * lds.E) = f32x4{0.f, 0.f, 0.f, 0.f};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (bits != 0) sm.tile(lds, at, at + TILE, qf, bits, lane);
        stage = stage + 1 == NS ? 0 : stage + 1;
    }
    sm.finish();
    __syncthreads();                        // the rings are done with
    float* o = reinterpret_cast<float*>(smem);                            // [waves][32 rows][PITCH]
    f32x4* ml = reinterpret_cast<f32x4*>(o + NW * 32 * F::PITCH);         // [waves][32]
    store_col<float, DB>(o + (wave * 32 + r) * F::PITCH, sm.acc, 1.f, DP, lane);
    if (lane < 32) ml[wave * 32 + r] = f32x4{sm.m, sm.sum, sm.rsum, 0.f};
    __syncthreads();
    for (int e = threadIdx.x; e < R * (a.D / 4); e += 64 * NW) {
        const int row = e / (a.D / 4), d = e % (a.D / 4) * 4;
        float m = NEG, sum = 0.f, rsum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[w * 32 + row][0]);
        const float mm = m == NEG ? 0.f : m;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const f32x4 t = ml[w * 32 + row], x = *reinterpret_cast<const f32x4*>(o + (w * 32 + row) * F::PITCH + d);
            const float f = __builtin_amdgcn_exp2f(t[0] - mm);
            sum = fmaf(t[1], f, sum);
            rsum = fmaf(t[2], f, rsum);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = fmaf(x[c], f, v[c]);
        }
        const int hh = job.hk * a.G + row % a.G;
        const int64_t to = ((int64_t)job.n * a.L + row / a.G) * a.H + hh, at = ((int64_t)job.n * a.H + hh) * a.L + row / a.G;
        if (a.splits > 1) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.o[0]) + split * a.numel + to * a.D + d) = v;
            if (d == 0) a.ml[(int64_t)split * a.N * a.H * a.L + at] = f32x4{m, sum, rsum, 0.f};
        } else {
            const float f = inverse(rsum), t[4] = {v[0] * f, v[1] * f, v[2] * f, v[3] * f};
            dfsfm::store_f32<T, 4>(static_cast<T*>(a.o[0]) + to * a.D + d, 4, t);
            if (d == 0) a.lse[at] = log_sum(m, sum);
        }
    }
}

// Joins up to FEW_SPLITS forward partials: 8 lanes a row, 4 channels a step, the splits added in their order, all loads under way before the
// first is used.  76800 rows x 3 splits x 32: 10 us (39 with a wave a row); 128 rows x 4 x 64: 4 us (6 with each split's load waited for).
constexpr int FEW_SPLITS = 8;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_few_kernel(const Attn a) {
    const int64_t rows = (int64_t)a.N * a.L * a.H, row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    if (row >= rows) return;
    const int h = (int)(row % a.H);
    const int64_t nl = row / a.H, at = (nl / a.L * a.H + h) * a.L + nl % a.L;
    f32x4 w[FEW_SPLITS];
    float m = NEG, sum = 0.f, rsum = 0.f;
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {          // all loads under way before the first is used
        w[s] = f32x4{NEG, 0.f, 0.f, 0.f};
        if (s < a.splits) w[s] = a.ml[s * rows + at];
    }
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) m = fmaxf(m, w[s][0]);
    const float mm = m == NEG ? 0.f : m;
#pragma unroll
    for (int s = 0; s < FEW_SPLITS; ++s) {
        w[s][0] = __builtin_amdgcn_exp2f(w[s][0] - mm);
        sum = fmaf(w[s][1], w[s][0], sum);
        rsum = fmaf(w[s][2], w[s][0], rsum);
    }
    const float inv = inverse(rsum);
    const float* part = static_cast<const float*>(a.o[0]) + row * a.D;
    for (int d = (threadIdx.x & 7) * 4; d < a.D; d += 32) {
        f32x4 t[FEW_SPLITS];
#pragma unroll
        for (int s = 0; s < FEW_SPLITS; ++s) {
            t[s] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (s < a.splits) t[s] = *reinterpret_cast<const f32x4*>(part + s * a.numel + d);
        }
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < FEW_SPLITS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(t[s][e], w[s][0] * inv, o[e]);
        dfsfm::store_f32<T, 4>(static_cast<T*>(a.o[1]) + row * a.D + d, 4, o);
    }
    if ((threadIdx.x & 7) == 0) a.lse[at] = log_sum(m, sum);
}

// Joins more of them, a wave a row: the lanes share the splits' maxima and sums, then 4 channels and every SG-th split each.
constexpr int MAX_SPLITS = 256;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const Attn a) {
    __shared__ float weight[4][MAX_SPLITS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t rows = (int64_t)a.N * a.L * a.H, row = (int64_t)blockIdx.x * 4 + wave, at0 = min(row, rows - 1);
    const int h = (int)(at0 % a.H);
    const int64_t nl = at0 / a.H, at = (nl / a.L * a.H + h) * a.L + nl % a.L;
    const f32x4* ml = a.ml + at;
    f32x4 v[MAX_SPLITS / 64];
    float m = NEG, sum = 0.f, rsum = 0.f;
#pragma unroll
    for (int i = 0; i < MAX_SPLITS / 64; ++i) {
        const int s = lane + 64 * i;
        v[i] = s < a.splits ? ml[s * rows] : f32x4{NEG, 0.f, 0.f, 0.f};
        m = fmaxf(m, v[i][0]);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mm = m == NEG ? 0.f : m;
#pragma unroll
    for (int i = 0; i < MAX_SPLITS / 64; ++i) {
        v[i][0] = __builtin_amdgcn_exp2f(v[i][0] - mm);
        sum = fmaf(v[i][1], v[i][0], sum);
        rsum = fmaf(v[i][2], v[i][0], rsum);
        weight[wave][lane + 64 * i] = v[i][0];
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        sum += __shfl_xor(sum, o);
        rsum += __shfl_xor(rsum, o);
    }
    __syncthreads();
    if (row >= rows) return;
    const int lanes = a.D <= 32 ? 8 : a.D <= 64 ? 16 : 32, d = lane % lanes * 4;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (d < a.D)
#pragma unroll 4
        for (int s = lane / lanes; s < a.splits; s += 64 / lanes) {
            const float f = weight[wave][s];
            const f32x4 t = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.o[0]) + s * a.numel + row * a.D + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(t[e], f, o[e]);
        }
    const float inv = inverse(rsum);
    for (int x = lanes; x < 64; x <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    if (d < a.D && lane < lanes) dfsfm::store_f32<T, 4>(static_cast<T*>(a.o[1]) + row * a.D + d, 4, o);
    if (lane == 0) a.lse[at] = log_sum(m, sum);
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
// delta: GIVEN, or summed here from p dp over the keys, which it is equal to.  The sum over the channels of dout times the ROUNDED out is off
// by half a step of out, an error that all keys of a row share: over many keys it drowns in the roundings of ds, over few it does not (dq of
// 4800 x 77 fp16: 3.2e-4 off in the 2-norm, 2.9e-4 so, 2.1e-4 by the output's rounding alone).  Two of three products are then made twice;
// up to two tiles of keys stay in LDS (RESIDENT: a pass over dout and out is saved), up to EXACT_KEYS keys are read TWICE.  Where delta is
// GIVEN and yet the keys may be few (a mask, up to FINE_KEYS of them, or one tile of rows), ds enters as two operands: dq of 248 rows x 7935
// keys, a tenth of them there, bf16 2.6e-3 -> 1.8e-3 off (1.7e-3 by the output's rounding alone); 4 x 4800 x 4800 x 8 x 32 with a mask,
// forward and gradient, 636 -> 687 us.
template <bool B>
struct Constant { static constexpr bool value = B; };
enum Delta { GIVEN, RESIDENT, TWICE };
constexpr int EXACT_KEYS = 512, FINE_KEYS = 2048;
template <typename T, int DP, Delta DELTA, bool FINE>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void attn_dq_kernel(const Attn a) {
    constexpr int DB = DP / 32, KS = DP / 16, TILE = Lds<T, DP>::TILE, KT = ROWS<T, DP>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Elem<T>* ks = reinterpret_cast<Elem<T>*>(smem);
    Elem<T>* vs = ks + 2 * TILE;
    const Job job(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Lds<T, DP> lds(lane);
    const int R = a.L * a.G, r = job.tile * 128 + wave * 32 + (lane & 31);
    const int l = r / a.G, h = job.hk * a.G + r % a.G;
    const int len = valid_len(a, job.n);
    const int per = ((len + KT - 1) / KT + a.splits - 1) / a.splits * KT;
    const int beg = min(len, job.split * per), end = min(len, beg + per);

    Frag<T> qf[KS], of[KS];
    const Mem<T>* qp = static_cast<const Mem<T>*>(a.q.p) + job.n * a.q.n + (int64_t)min(l, a.L - 1) * a.q.l + h * a.q.h;
    const Mem<T>* op = static_cast<const Mem<T>*>(a.dout.p) + job.n * a.dout.n + (int64_t)min(l, a.L - 1) * a.dout.l + h * a.dout.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * (lane >> 5);
        qf[s] = r < R && c < a.D ? load8<T>(qp + c) : zero_frag<T>();
        of[s] = r < R && c < a.D ? load8<T>(op + c) : zero_frag<T>();
    }
    const int64_t at = ((int64_t)job.n * a.H + h) * a.L + l;
    const float c = a.scale * LOG2E, lse = r < R ? a.lse[at] : NEG;
    const float lse2 = lse == NEG ? INFINITY : lse * LOG2E;              // a row without keys has p = 0
    float delta = DELTA == GIVEN && r < R ? a.delta[at] : 0.f;
    const Elem<T>* kb = static_cast<const Elem<T>*>(a.kt.p) + job.n * a.kt.n + job.hk * a.kt.h;
    const Elem<T>* vb = static_cast<const Elem<T>*>(a.vt.p) + job.n * a.vt.n + job.hk * a.vt.h;
    const Dma<T, DP, KT, 256> dk(a.kt.l, a.D, a.plane_k), dv(a.vt.l, a.D, a.plane_k);
    unsigned mask = 0;
    auto fetch = [&](int s0, int buf) {
        dk.issue(kb + s0 * a.kt.l, end - s0, ks + buf * TILE);
        dv.issue(vb + s0 * a.vt.l, end - s0, vs + buf * TILE);
        mask = key_mask(a, job.n, s0);
    };
    // keys that the mask drops: p is 0, which does not undo a NaN in dp or k
    auto clear = [&](int buf, unsigned long long bits) {
        if (a.mask && bits != ALL_KEYS<KT> && bits) {
            zero_rows<T, DP>(ks + buf * TILE, bits);
            zero_rows<T, DP>(vs + buf * TILE, bits);
            __syncthreads();
        }
    };
    f32x16 acc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) acc[b] = splat16(0.f);
    ColumnScale<T, DB> cs;
    // p dp of 32 keys, dp less delta
    auto products = [&](int buf, int b, unsigned long long bits, f32x16& ds) {
        const Elem<T>* kt = ks + buf * TILE;
        const Elem<T>* vt = vs + buf * TILE;
        f32x16 st = splat16(0.f);
        ds = splat16(-delta);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            st = Mma<T>::run(lds.read_rows(kt, 32 * b, 16 * s), qf[s], st);
            ds = Mma<T>::run(lds.read_rows(vt, 32 * b, 16 * s), of[s], ds);
        }
        if (bits != ALL_KEYS<KT>) drop_keys(st, (unsigned)(bits >> 32 * b >> 4 * (lane >> 5)));
#pragma unroll
        for (int j = 0; j < 16; ++j) ds[j] *= __builtin_amdgcn_exp2f(fmaf(st[j], c, -lse2));
    };
    auto accumulate = [&](auto fine, int buf, unsigned long long bits) {
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
            if (b && bits >> 32 == 0) break;
            f32x16 ds[1];
            products(buf, b, bits, ds[0]);
            cs.apply(ds, acc);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Operand<T, decltype(fine)::value> p(ds[0], u);
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = p.times(lds.read_cols(ks + buf * TILE, 32 * b + 16 * u, 32 * d), acc[d]);
            }
        }
    };
    typedef Constant<FINE> Chosen;
    if constexpr (DELTA != GIVEN) {
        float sum = 0.f;
        auto add = [&](int buf, unsigned long long bits) {
            for (int b = 0; b < KT / 32; ++b) {
                if (b && bits >> 32 == 0) break;
                f32x16 ds;
                products(buf, b, bits, ds);
#pragma unroll
                for (int j = 0; j < 16; ++j) sum += ds[j];
            }
        };
        auto added = [&]() {
            delta = dfsfm::add_xor32(sum);
            if (r < R && lane < 32) a.delta[at] = delta;
        };
        if constexpr (DELTA == RESIDENT) {
            unsigned long long bits[2] = {0, 0};
            unsigned masks[2] = {0, 0};
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (t * KT < end) {
                    fetch(t * KT, t);
                    masks[t] = mask;
                }
            dma_landed();
#pragma unroll
            for (int t = 0; t < 2; ++t) bits[t] = key_bits<KT>(masks[t], t * KT, end);
            __syncthreads();
            clear(0, bits[0]);
            clear(1, bits[1]);
            for (int t = 0; t * KT < end; ++t)
                if (bits[t]) add(t, bits[t]);
            added();
            for (int t = 0; t * KT < end; ++t)
                if (bits[t]) accumulate(Chosen(), t, bits[t]);
        } else {
            const int tiles = (end + KT - 1) / KT;
            if (tiles) fetch(0, 0);
            else added();
            for (int i = 0; i < 2 * tiles; ++i) {
                const int s0 = (i < tiles ? i : i - tiles) * KT, buf = i & 1;
                dma_landed();
                const unsigned long long bits = key_bits<KT>(mask, s0, end);
                __syncthreads();
                clear(buf, bits);
                if (i + 1 < 2 * tiles) fetch((i + 1 < tiles ? i + 1 : i + 1 - tiles) * KT, buf ^ 1);
                if (i == tiles) added();
                if (bits && i < tiles) add(buf, bits);
                if (bits && i >= tiles) accumulate(Chosen(), buf, bits);
            }
        }
    } else {
        auto walk = [&](auto fine) {
            if (beg < end) fetch(beg, 0);
            int buf = 0;
            for (int s0 = beg; s0 < end; s0 += KT, buf ^= 1) {
                dma_landed();
                const unsigned long long bits = key_bits<KT>(mask, s0, end);
                __syncthreads();
                clear(buf, bits);
                if (s0 + KT < end) fetch(s0 + KT, buf ^ 1);
                if (bits && job.tile * 128 + wave * 32 < R) accumulate(fine, buf, bits);
            }
        };
        if (ROUNDS<T> && !FINE && (a.mask || len <= FINE_KEYS))
            walk(Constant<ROUNDS<T>>());
        else
            walk(Chosen());
    }
    if (r >= R) return;
    const int64_t row = ((int64_t)job.n * a.L + l) * a.H + h;
    const float f = a.scale / cs.f;
    if (a.splits > 1)
        store_col<float, DB>(static_cast<float*>(a.o[0]) + job.split * a.numel + row * a.D, acc, f, a.D, lane);
    else
        store_col<Mem<T>, DB>(static_cast<Mem<T>*>(a.o[0]) + row * a.D, acc, f, a.D, lane);
}

// dk and dv: NW waves x 32 keys a workgroup, tiles of 64 rows of q and dout, both read both ways.
//
// NW is 4, two workgroups a CU, where a wave's K, V, dk and dv leave room for two waves a SIMD.  At D = 128 in 16 bits they are 192 registers
// before the first score; there NW is 8, one workgroup a CU, and V stays in LDS (64 KB for 256 keys), read again for every tile.
// 4 x 4800 x 6400 (ragged) x 16 heads bf16 takes 1.10 - 1.19 ms; with V in registers, four waves and one wave a SIMD 2.3; with the two halves
// of the work on two waves that pass p through LDS 1.7; as two launches, one product made twice, 1.8.
template <typename T, int DP>
constexpr int KEY_WAVES = DP == 128 && sizeof(Mem<T>) == 2 ? 8 : 4;

template <typename T, int DP, bool FINE>
__global__ __launch_bounds__((64 * KEY_WAVES<T, DP>), (KEY_WAVES<T, DP> / 4)) void attn_dkdv_kernel(const Attn a) {
    constexpr int NW = KEY_WAVES<T, DP>, THREADS = 64 * NW;
    constexpr bool VLDS = NW == 8;
    constexpr int UNROLL = VLDS ? 1 : 2;
    constexpr int DB = DP / 32, KS = DP / 16, TILE = Lds<T, DP>::TILE, KT = ROWS<T, DP>;
    // p of fp16 tensors times 2^14: a power of two that keeps weights down to 2^-28 exact and 1 in range
    constexpr float SHIFT = __is_same(T, f16) ? 14.f : 0.f, UNSHIFT = __is_same(T, f16) ? 1.f / 16384.f : 1.f;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Elem<T>* qs = reinterpret_cast<Elem<T>*>(smem);
    Elem<T>* os = qs + 2 * TILE;
    Elem<T>* vs = os + 2 * TILE;                                                // VLDS: the workgroup's keys
    float* rowv = reinterpret_cast<float*>(vs + (VLDS ? NW * 32 * DP : 0));      // [2][2][64]: -lse / scale, -delta
    const Job job(a, a.tiles, a.splits, NW * 32);
    // which of the workgroup's keys a wave has turns with the workgroup: waves without any are not all on one SIMD
    const int lane = threadIdx.x & 63, wave = ((threadIdx.x >> 6) + blockIdx.x) % NW, hkv = a.H / a.G;
    const Lds<T, DP> lds(lane);
    const int s = job.tile * (NW * 32) + wave * 32 + (lane & 31);
    const int len = valid_len(a, job.n);
    bool there = s < len;
    if (a.mask) there = there && a.mask[(int64_t)job.n * a.S + min(s, a.S - 1)] != 0;
    // a tile is 64 queries of one of the G heads; splits take whole tiles
    const int lt = (a.L + KT - 1) / KT, per = (lt * a.G + a.splits - 1) / a.splits;
    const int beg = min(lt * a.G, job.split * per), end = min(lt * a.G, beg + per);

    Frag<T> kf[KS], vf[VLDS ? 1 : KS];
    const Mem<T>* kp = static_cast<const Mem<T>*>(a.k.p) + job.n * a.k.n + (int64_t)min(s, a.S - 1) * a.k.l + job.hk * a.k.h;
    const Mem<T>* vp = static_cast<const Mem<T>*>(a.v.p) + job.n * a.v.n + (int64_t)min(s, a.S - 1) * a.v.l + job.hk * a.v.h;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
        const int c = 16 * x + 8 * (lane >> 5);
        kf[x] = there && c < a.D ? load8<T>(kp + c) : zero_frag<T>();
        if constexpr (!VLDS) vf[x] = there && c < a.D ? load8<T>(vp + c) : zero_frag<T>();
    }
    const Elem<T>* qb = static_cast<const Elem<T>*>(a.qt.p) + job.n * a.qt.n + job.hk * a.G * a.qt.h;
    const Elem<T>* ob = static_cast<const Elem<T>*>(a.dt.p) + job.n * a.dt.n + job.hk * a.G * a.dt.h;
    const int64_t vec = ((int64_t)job.n * a.H + job.hk * a.G) * a.L;
    const Dma<T, DP, KT, THREADS> dq(a.qt.l, a.D, a.plane_q), dd(a.dt.l, a.D, a.plane_q);
    float rv = 0.f;                         // threads below KT: lse of a row, the next KT: delta
    const float inv_scale = 1.f / a.scale;
    int rows = 0;                           // rows of the tile in flight
    auto fetch = [&](int it, int buf) {
        const int g = it / lt, l0 = (it - g * lt) * KT;
        rows = a.L - l0;
        dq.issue(qb + g * a.qt.h + l0 * a.qt.l, rows, qs + buf * TILE);
        dd.issue(ob + g * a.dt.h + l0 * a.dt.l, rows, os + buf * TILE);
        if (threadIdx.x < 2 * KT) {
            const int row = threadIdx.x % KT;
            rv = (threadIdx.x < KT ? a.lse : a.delta)[vec + (int64_t)g * a.L + l0 + min(row, rows - 1)];
        }
    };
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) dk[b] = dv[b] = splat16(0.f);
    ColumnScale<T, DB> cs;
    const float c = a.scale * LOG2E;
    const bool any = __syncthreads_or(there);
    if (any && beg < end) {
        if constexpr (VLDS) {               // masked keys come as they are: a key's column is its own, and dropped at the end
            const int s0 = job.tile * (NW * 32);
            const Dma<T, DP, NW * 32, THREADS> dv(a.vt.l, a.D, a.plane_k);
            dv.issue(static_cast<const Elem<T>*>(a.vt.p) + job.n * a.vt.n + job.hk * a.vt.h + s0 * a.vt.l, len - s0, vs);
        }
        fetch(beg, 0);
    }
    // Behind the first fetch, which the loop waits for at once.  2 x 4800 x 4800 x 8 x 64 bf16 forward and gradient 562 -> 557 us, x 128 fp16
    // 1108 -> 1104.  Unsettled, D = 32 (130 us, 132 settled) and two operands (16 tokens x 10816 x 8 x 64: 176, 178) do a little better.
    if constexpr (ROUNDS<T> && DP >= 64 && !FINE) {
        settle<T>(kf);
        if constexpr (!VLDS) settle<T>(vf);
    }
    const bool mine = __ballot(there) != 0;
    int buf = 0;
    for (int it = beg; any && it < end; ++it, buf ^= 1) {
        const Elem<T>* qt = qs + buf * TILE;
        const Elem<T>* ot = os + buf * TILE;
        float* vt = rowv + buf * 2 * KT;
        dma_landed();
        // -lse / scale and -delta start the sums; a row without keys, or behind the last, gets a score of -inf: p = 0
        if (threadIdx.x < 2 * KT) {
            const bool in = (int)(threadIdx.x % KT) < rows;
            vt[threadIdx.x] = threadIdx.x < KT ? (in && rv != NEG ? -rv * (ROUNDS<T> ? inv_scale : LOG2E) : NEG) : (in ? -rv : 0.f);
        }
        __syncthreads();
        if (it + 1 < end) fetch(it + 1, buf ^ 1);
        if (!mine) continue;
#pragma unroll UNROLL
        for (int b = 0; b < KT / 32; ++b) {
            f32x16 st = ROUNDS<T> ? rows16(vt + 32 * b, lane) : splat16(0.f);
            f32x16 ds[1];
            ds[0] = rows16(vt + KT + 32 * b, lane);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                st = Mma<T>::run(lds.read_rows(qt, 32 * b, 16 * x), kf[x], st);
                ds[0] = Mma<T>::run(lds.read_rows(ot, 32 * b, 16 * x), VLDS ? lds.read_rows(vs, 32 * wave, 16 * x) : vf[VLDS ? 0 : x], ds[0]);
            }
            // 32 bits: the sums start at 0 and lse is taken off at the end, in one rounding
            const f32x16 off = ROUNDS<T> ? splat16(SHIFT) : rows16(vt + 32 * b, lane);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                st[j] = __builtin_amdgcn_exp2f(fmaf(st[j], c, off[j]));
                ds[0][j] *= st[j];
            }
            cs.apply(ds, dk);
            if constexpr (VLDS) __builtin_amdgcn_sched_barrier(0);       // with the loop above not unrolled: no register spilled
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Operand<T, FINE> p(st, u), g(ds[0], u);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    dv[d] = p.times(lds.read_cols(ot, 32 * b + 16 * u, 32 * d), dv[d]);
                    dk[d] = g.times(lds.read_cols(qt, 32 * b + 16 * u, 32 * d), dk[d]);
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
        store_col<Mem<T>, DB>(static_cast<Mem<T>*>(a.o[0]) + row * a.D, dk, f, a.D, lane);
        store_col<Mem<T>, DB>(static_cast<Mem<T>*>(a.o[1]) + row * a.D, dv, UNSHIFT, a.D, lane);
    }
}

// x = sum of the splits' partials, in their order; blockIdx.y 1: y, from the partials behind
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* __restrict__ part, int64_t numel, int splits, T* __restrict__ x, T* __restrict__ y) {
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;      // D is a multiple of 8, so numel is
    if (e >= numel) return;
    part += blockIdx.y * splits * numel + e;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) o += *reinterpret_cast<const f32x4*>(part + s * numel);
    const float t[4] = {o[0], o[1], o[2], o[3]};
    dfsfm::store_f32<T, 4>((blockIdx.y ? y : x) + e, 4, t);
}

// The three planes of x (blockIdx.y 0) or y (1), [N, len, heads, D] fp32, dense: 8 channels a thread.
__global__ __launch_bounds__(256) void attn_planes_kernel(const Tensor x, const Tensor y, int len, int heads, int D, bf16* __restrict__ to, int64_t plane) {
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (e >= plane) return;
    const Tensor& t = blockIdx.y ? y : x;
    const int64_t row = e / D, nl = row / heads;
    const Frag3 f = load8<X3>(static_cast<const float*>(t.p) + nl / len * t.n + nl % len * t.l + row % heads * t.h + e % D);
    bf16* o = to + (blockIdx.y ? 3 * plane : 0) + e;
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(o + k * plane) = f.p[k];
}

// ---------------------------------------------------------------- host
int pad_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// 1 / scale and scale * log2(e) are 32-bit numbers
bool scale_ok(float s) { return s >= 1e-20f && s <= 1e20f; }

// 16-byte loads; offsets within a tile of 64 rows are 32-bit byte offsets; a row does not overlap the next
bool rows_ok(const void* p, int64_t n, int64_t l, int64_t h, int D, int dtype) {
    const int64_t e = dtype == DFSFM_F32 ? 4 : 8;
    return !((uintptr_t)p & 15) && n % e == 0 && l % e == 0 && h % e == 0 && l >= D && l < (1ll << 23);
}

// Splits of the long axis (`length` rows of it, `least` a split).  `slots` workgroups run at a time (512: two a CU; of instances that leave
// room for one, two rounds); as long as they number less than eight such rounds the last one's idle places count, and the smallest number of
// splits that fills 85 % of the places is taken: 608 workgroups of the forward pass 2 x 4800 x 10816 x 8 x 32 fp32 take 637 us, three splits of
// each 530 - 570 with planes and join.
// A join is 5 us, what 256 keys of 16 bits take a wave; of fp32's products (32 keys of 128 channels: 3 us in planes, 5 on the 32-bit
// instruction) 64 keys are worth one: 33 x 1387 x 4 x 80 forward and gradient 140 -> 81 us, one row of 4 x 3271 keys 120 -> 76.
int choose_splits(int64_t groups, int64_t length, int slots, int least) {
    if (groups <= 0 || groups >= 8 * slots) return 1;
    const int64_t most = length / least < MAX_SPLITS ? length / least : MAX_SPLITS;
    int best = 1;
    double fill = 0;
    for (int s = 1; s <= most || s == 1; ++s) {
        const int64_t n = groups * s, places = (n + slots - 1) / slots * slots;
        const double f = (double)n / (double)places;
        if (f > fill * 1.02) fill = f, best = s;
        if (fill >= 0.85) break;
    }
    return best;
}

// The launches of a call, from its sizes alone.
struct Plan {
    int heads, tq, tk, fwd, dq, dkdv;       // row tiles, key tiles, splits
    bool few, xq, xk;                            // fp32 in three planes: the kernels that walk the keys, the one that walks the rows
    int64_t rows, keys;                     // elements of q (or out), of k
    Plan(int N, int L, int S, int H, int Hkv, int D, int dtype) {
        heads = N * Hkv;
        const int64_t R = (int64_t)L * (H / Hkv);
        // Planes of k and v (or of q and dout) cost 20 bytes an element and pay from 64 rows (or keys) a head on; fewer are bound by memory.
        xq = dtype == DFSFM_F32 && R > 64;
        xk = dtype == DFSFM_F32 && S > 64;
        const int wave_keys = 32 * (dtype != DFSFM_F32 && pad_dim(D) == 128 ? KEY_WAVES<bf16, 128> : KEY_WAVES<bf16, 32>);
        const int least = dtype == DFSFM_F32 ? 64 : 256;
        tq = (int)((R + 127) / 128);
        tk = (S + wave_keys - 1) / wave_keys;
        few = R <= 32;
        // Few rows read their keys once, from memory: about a workgroup a CU does without the join (256 heads x 8192 x 64 fp16: 98 us against
        // 110 in two splits, x 128 bf16 178 and 186), below that two a CU (128 heads x 10816 ragged keys x 64: 53 us in four splits, 68 in two,
        // 54 in eight; x 128 bf16 95, 91 and 87, x 32 45, 43 and 35).
        fwd = few && heads >= 200 ? 1 : choose_splits((int64_t)heads * tq, S, tq == 1 && !few ? 2048 : 512, least);
        dq = S <= (dtype == DFSFM_F32 ? 128 : EXACT_KEYS) ? 1 : choose_splits((int64_t)heads * tq, S, tq == 1 ? 2048 : 512, least);
        dkdv = choose_splits((int64_t)heads * tk, R, wave_keys == 256 ? 256 : 512, least);
        rows = (int64_t)N * L * H * D;
        keys = (int64_t)N * S * Hkv * D;
    }
    // bytes of workspaces
    size_t planes_k() const { return xq ? (size_t)keys * 12 : 0; }
    size_t planes_q() const { return xk ? (size_t)rows * 12 : 0; }
    size_t forward(int D) const { return planes_k() + (fwd > 1 ? (size_t)fwd * (rows + rows / D * 4) * 4 : 0); }
    size_t delta(int D) const { return ((size_t)(rows / D) * 4 + 15) / 16 * 16; }
    size_t backward(int D) const {
        const size_t a = planes_k() + (dq > 1 ? (size_t)dq * rows * 4 : 0), b = planes_q() + (dkdv > 1 ? (size_t)2 * dkdv * keys * 4 : 0);
        return delta(D) + (a > b ? a : b);
    }
};

bool shape_ok(int N, int L, int S, int H, int Hkv, int D, bool backward) {
    if (D <= 0 || D > 128 || D % 8 || Hkv <= 0 || H % Hkv || (int64_t)H * D >= (1 << 23)) return false;
    const int64_t R = (int64_t)L * (H / Hkv), heads = (int64_t)N * Hkv, tq = (R + 127) / 128, tk = ((int64_t)S + 127) / 128;
    // row and workgroup numbers are 32-bit
    if (R >= (1ll << 30) || S >= (1 << 30) || heads >= (1 << 20) || heads * (tq + 2048) >= (1ll << 31) || heads * (tk + 2048) >= (1ll << 31)) return false;
    // a launch holds less than 2^32 threads along an axis: of the attention kernels 256 a tile of 128 rows or keys, of delta's 8 a row (of the
    // planes' one for 8 values: 2^32 of them have planes of 412 GB, more than there is)
    return heads * tq < (1 << 24) && heads * tk < (1 << 24) && (!backward || heads * R < (1ll << 29));
}

// The planes of two tensors of the same sizes, dense, at `to`; the tensors as tiles are fetched from them.
void make_planes(const Tensor& x, const Tensor& y, int N, int len, int heads, int D, void* to, Tensor& xt, Tensor& yt, int64_t& plane, hipStream_t st) {
    plane = (int64_t)N * len * heads * D;
    bf16* p = static_cast<bf16*>(to);
    xt = {p, (int64_t)len * heads * D, (int64_t)heads * D, D};
    yt = {p + 3 * plane, (int64_t)len * heads * D, (int64_t)heads * D, D};
    if (plane > 0)
        hipLaunchKernelGGL(attn_planes_kernel, dim3((unsigned)((plane / 8 + 255) / 256), 2), dim3(256), 0, st, x, y, len, heads, D, p, plane);
}

template <typename T, int DP>
int forward_dp(Attn a, const Plan& p, void* out, hipStream_t st) {
    constexpr int smem = 4 * Lds<T, DP>::TILE * sizeof(Elem<T>);
    static dfsfm::SmemAttr attr;
    attr.ensure(reinterpret_cast<const void*>(&attn_forward_kernel<T, DP>), smem);
    a.tiles = p.tq;
    a.splits = p.fwd;
    if (p.fwd == 1) a.o[0] = out;
    const dim3 grid((unsigned)(p.heads * p.tq * p.fwd));
    bool done = false;
    if constexpr (!__is_same(T, X3)) {
        if (p.few) {
            typedef Few<T, DP> F;
            static dfsfm::SmemAttr few;
            few.ensure(reinterpret_cast<const void*>(&attn_forward_few_kernel<T, DP>), F::SMEM);
            hipLaunchKernelGGL((attn_forward_few_kernel<T, DP>), grid, dim3(64 * F::WAVES), F::SMEM, st, a);
            done = true;
        }
    }
    if (!done) hipLaunchKernelGGL((attn_forward_kernel<T, DP>), grid, dim3(256), smem, st, a);
    if (p.fwd > 1) {
        a.o[1] = out;
        const int64_t rows = (int64_t)a.N * a.L * a.H;
        if (p.fwd <= FEW_SPLITS)
            hipLaunchKernelGGL((attn_join_few_kernel<Mem<T>>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((attn_join_kernel<Mem<T>>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    }
    return check_launch("dfsfm_cross_attention");
}

template <typename T, int DP>
int dq_dp(Attn a, const Plan& p, Mem<T>* dq, float* part, hipStream_t st) {
    typedef Mem<T> M;
    const int64_t rows = p.rows / a.D;
    constexpr int smem = 4 * Lds<T, DP>::TILE * sizeof(Elem<T>);
    a.tiles = p.tq;
    a.splits = p.dq;
    a.numel = p.rows;
    a.o[0] = p.dq > 1 ? static_cast<void*>(part) : dq;
    const dim3 grid((unsigned)(p.heads * p.tq * p.dq));
    auto launch = [&](auto kernel, dfsfm::SmemAttr& attr) {
        attr.ensure(reinterpret_cast<const void*>(kernel), smem);
        hipLaunchKernelGGL(kernel, grid, dim3(256), smem, st, a);
    };
    static dfsfm::SmemAttr attr[6];
    const bool fine = ROUNDS<T> && p.tq == 1;
    if (a.S <= 2 * ROWS<T, DP>) {
        if (fine)
            launch(&attn_dq_kernel<T, DP, RESIDENT, ROUNDS<T>>, attr[0]);
        else
            launch(&attn_dq_kernel<T, DP, RESIDENT, false>, attr[1]);
    } else if (ROUNDS<T> && a.S <= EXACT_KEYS) {
        constexpr Delta HOW = ROUNDS<T> ? TWICE : GIVEN;
        if (fine)
            launch(&attn_dq_kernel<T, DP, HOW, ROUNDS<T>>, attr[2]);
        else
            launch(&attn_dq_kernel<T, DP, HOW, false>, attr[3]);
    } else {
        hipLaunchKernelGGL((attn_delta_kernel<M>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, st, a);
        if (fine)
            launch(&attn_dq_kernel<T, DP, GIVEN, ROUNDS<T>>, attr[4]);
        else
            launch(&attn_dq_kernel<T, DP, GIVEN, false>, attr[5]);
    }
    if (p.dq > 1)
        hipLaunchKernelGGL((attn_sum_kernel<M>), dim3((unsigned)((p.rows / 4 + 255) / 256)), dim3(256), 0, st, part, p.rows, p.dq, dq, dq);
    return check_launch("dfsfm_cross_attention_backward");
}

template <typename T, int DP>
int dkdv_dp(Attn a, const Plan& p, Mem<T>* dk, Mem<T>* dv, float* part, hipStream_t st) {
    typedef Mem<T> M;
    a.tiles = p.tk;
    a.splits = p.dkdv;
    a.numel = p.keys;
    a.o[0] = p.dkdv > 1 ? static_cast<void*>(part) : dk;
    a.o[1] = p.dkdv > 1 ? static_cast<void*>(part + p.dkdv * p.keys) : dv;
    constexpr int NW = KEY_WAVES<T, DP>;
    constexpr int smem = (4 * Lds<T, DP>::TILE + (NW == 8 ? NW * 32 * DP : 0)) * sizeof(Elem<T>) + 4 * ROWS<T, DP> * 4;
    const dim3 grid((unsigned)(p.heads * p.tk * p.dkdv));
    if (ROUNDS<T> && (p.few || a.S <= 32)) {
        static dfsfm::SmemAttr attr;
        attr.ensure(reinterpret_cast<const void*>(&attn_dkdv_kernel<T, DP, ROUNDS<T>>), smem);
        hipLaunchKernelGGL((attn_dkdv_kernel<T, DP, ROUNDS<T>>), grid, dim3(64 * NW), smem, st, a);
    } else {
        static dfsfm::SmemAttr attr;
        attr.ensure(reinterpret_cast<const void*>(&attn_dkdv_kernel<T, DP, false>), smem);
        hipLaunchKernelGGL((attn_dkdv_kernel<T, DP, false>), grid, dim3(64 * NW), smem, st, a);
    }
    if (p.dkdv > 1) {
        hipLaunchKernelGGL((attn_sum_kernel<M>), dim3((unsigned)((p.keys / 4 + 255) / 256), 2), dim3(256), 0, st, part, p.keys, p.dkdv, dk, dv);
    }
    return check_launch("dfsfm_cross_attention_backward");
}

// CALL with T the type `dtype` (fp32 in planes if `wide`) and DP the padded head dim
#define DFSFM_ATTN_DIM(CALL, T)                      \
    switch (pad_dim(a.D)) {                          \
        case 32: { constexpr int DP = 32; return CALL; }   \
        case 64: { constexpr int DP = 64; return CALL; }   \
        default: { constexpr int DP = 128; return CALL; }  \
    }
#define DFSFM_ATTN_CALL(dtype, wide, CALL)                              \
    if (dtype == DFSFM_BF16) { typedef bf16 T; DFSFM_ATTN_DIM(CALL, T) } \
    if (dtype == DFSFM_F16) { typedef f16 T; DFSFM_ATTN_DIM(CALL, T) }   \
    if (wide) { typedef X3 T; DFSFM_ATTN_DIM(CALL, T) }                  \
    { typedef float T; DFSFM_ATTN_DIM(CALL, T) }

int forward_any(const Attn& a, const Plan& p, int dtype, void* out, hipStream_t st) {
    DFSFM_ATTN_CALL(dtype, p.xq, (forward_dp<T, DP>(a, p, out, st)))
}
int dq_any(const Attn& a, const Plan& p, int dtype, void* dq, float* part, hipStream_t st) {
    DFSFM_ATTN_CALL(dtype, p.xq, (dq_dp<T, DP>(a, p, (Mem<T>*)dq, part, st)))
}
int dkdv_any(const Attn& a, const Plan& p, int dtype, void* dk, void* dv, float* part, hipStream_t st) {
    DFSFM_ATTN_CALL(dtype, p.xk, (dkdv_dp<T, DP>(a, p, (Mem<T>*)dk, (Mem<T>*)dv, part, st)))
}

}  // namespace

extern "C" size_t dfsfm_cross_attention_workspace(int N, int L, int S, int H, int Hkv, int D, int dtype) {
    if (N <= 0 || L <= 0 || S < 0 || H <= 0 || !shape_ok(N, L, S, H, Hkv, D, false)) return 0;
    return Plan(N, L, S, H, Hkv, D, dtype).forward(D);
}

extern "C" int dfsfm_cross_attention(const void* q, int64_t qn, int64_t ql, int64_t qh, const void* k, int64_t kn, int64_t ks, int64_t kh,
                                     const void* v, int64_t vn, int64_t vs, int64_t vh, const int* kv_lens, const uint8_t* kv_mask,
                                     void* out, float* lse, int N, int L, int S, int H, int Hkv, int D, float scale, int dtype,
                                     void* workspace, size_t workspace_bytes, void* stream_) {
    if (N == 0 || L == 0 || H == 0) return DFSFM_OK;
    if (!q || !out || !lse || (S > 0 && (!k || !v)) || N < 0 || L < 0 || S < 0 || H < 0 || !scale_ok(scale)) return DFSFM_E_BADARG;
    if (!shape_ok(N, L, S, H, Hkv, D, false)) return DFSFM_E_UNSUPPORTED;
    if (dtype < DFSFM_F32 || dtype > DFSFM_F16 || !rows_ok(q, qn, ql, qh, D, dtype) || ((uintptr_t)out & 15)) return DFSFM_E_UNSUPPORTED;
    if (S > 0 && (!rows_ok(k, kn, ks, kh, D, dtype) || !rows_ok(v, vn, vs, vh, D, dtype))) return DFSFM_E_UNSUPPORTED;
    const Plan p(N, L, S, H, Hkv, D, dtype);
    if (workspace_bytes < p.forward(D) || (p.forward(D) > 0 && (!workspace || ((uintptr_t)workspace & 15)))) return DFSFM_E_WORKSPACE;
    hipStream_t st = static_cast<hipStream_t>(stream_);
    Attn a{};
    a.q = {q, qn, ql, qh};
    a.k = a.kt = {k, kn, ks, kh};
    a.v = a.vt = {v, vn, vs, vh};
    a.lens = kv_lens;
    a.mask = kv_mask;
    a.lse = lse;
    a.N = N, a.L = L, a.S = S, a.H = H, a.G = H / Hkv, a.D = D, a.scale = scale;
    a.numel = p.rows;
    if (p.xq) make_planes(a.k, a.v, N, S, Hkv, D, workspace, a.kt, a.vt, a.plane_k, st);
    a.o[0] = static_cast<char*>(workspace) + p.planes_k();
    a.ml = reinterpret_cast<f32x4*>(static_cast<float*>(a.o[0]) + p.fwd * p.rows);
    return forward_any(a, p, dtype, out, st);
}

extern "C" size_t dfsfm_cross_attention_backward_workspace(int N, int L, int S, int H, int Hkv, int D, int dtype) {
    if (N <= 0 || L < 0 || S < 0 || H <= 0 || !shape_ok(N, L, S, H, Hkv, D, true)) return 0;
    return Plan(N, L, S, H, Hkv, D, dtype).backward(D);
}

extern "C" int dfsfm_cross_attention_backward(const void* dout, int64_t gn, int64_t gl, int64_t gh, const void* q, int64_t qn, int64_t ql,
                                              int64_t qh, const void* k, int64_t kn, int64_t ks, int64_t kh, const void* v, int64_t vn,
                                              int64_t vs, int64_t vh, const void* out, int64_t on, int64_t ol, int64_t oh, const float* lse,
                                              const int* kv_lens, const uint8_t* kv_mask, void* dq, void* dk, void* dv, int N, int L, int S,
                                              int H, int Hkv, int D, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                              void* stream_) {
    if (N == 0 || H == 0 || (L == 0 && S == 0)) return DFSFM_OK;
    if (N < 0 || L < 0 || S < 0 || H < 0 || !scale_ok(scale)) return DFSFM_E_BADARG;
    if ((L > 0 && (!dout || !q || !out || !lse || !dq)) || (S > 0 && (!k || !v || !dk || !dv))) return DFSFM_E_BADARG;
    if (!shape_ok(N, L, S, H, Hkv, D, true)) return DFSFM_E_UNSUPPORTED;
    if (dtype < DFSFM_F32 || dtype > DFSFM_F16 || (((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15)) return DFSFM_E_UNSUPPORTED;
    if (L > 0 && (!rows_ok(q, qn, ql, qh, D, dtype) || !rows_ok(dout, gn, gl, gh, D, dtype) || !rows_ok(out, on, ol, oh, D, dtype)))
        return DFSFM_E_UNSUPPORTED;
    if (S > 0 && (!rows_ok(k, kn, ks, kh, D, dtype) || !rows_ok(v, vn, vs, vh, D, dtype))) return DFSFM_E_UNSUPPORTED;
    const Plan p(N, L, S, H, Hkv, D, dtype);
    if (workspace_bytes < p.backward(D) || (p.backward(D) > 0 && (!workspace || ((uintptr_t)workspace & 15)))) return DFSFM_E_WORKSPACE;
    hipStream_t st = static_cast<hipStream_t>(stream_);
    Attn a{};
    a.q = a.qt = {q, qn, ql, qh};
    a.k = a.kt = {k, kn, ks, kh};
    a.v = a.vt = {v, vn, vs, vh};
    a.dout = a.dt = {dout, gn, gl, gh};
    a.out = {out, on, ol, oh};
    a.lens = kv_lens;
    a.mask = kv_mask;
    a.lse = const_cast<float*>(lse);
    a.N = N, a.L = L, a.S = S, a.H = H, a.G = H / Hkv, a.D = D, a.scale = scale;
    a.delta = static_cast<float*>(workspace);
    char* scratch = static_cast<char*>(workspace) + p.delta(D);            // dq's first, then the other's
    if (L > 0) {
        if (p.xq) make_planes(a.k, a.v, N, S, Hkv, D, scratch, a.kt, a.vt, a.plane_k, st);
        const int rc = dq_any(a, p, dtype, dq, reinterpret_cast<float*>(scratch + p.planes_k()), st);
        if (rc != DFSFM_OK) return rc;
    }
    if (S > 0) {
        a.kt = a.k, a.vt = a.v;
        if (p.xk) make_planes(a.q, a.dout, N, L, H, D, scratch, a.qt, a.dt, a.plane_q, st);
        return dkdv_any(a, p, dtype, dk, dv, reinterpret_cast<float*>(scratch + p.planes_q()), st);
    }
    return DFSFM_OK;
}
