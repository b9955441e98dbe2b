// Matrix products with a fused epilogue: y = act(x w^T + b) + r, and the two products of its backward
// (formulas: include/sparsemarg.h).  Compute bound on the matrix cores for many rows, bound by
// reading w for few.
//
// One kernel C[m][n] = sum_k A(m, k) B(n, k) serves all three: an operand is stored either with k
// consecutive ("rows": x and w in the forward) or with m (n) consecutive ("columns": w in dx = dh w,
// both in dw = dh^T x).  A row tile is staged as [m][k] and read 16 bytes per lane; a column tile is
// staged as it lies, [k][m], and transposed by the LDS read (ds_read_b64_tr_b16: 16 lanes read 4 k
// rows of 16 elements and each receives one column).  Both give a lane 8 consecutive k of one m,
// the operand layout of v_mfma_f32_16x16x32.  The product is computed as C^T tiles (B first), so that a
// lane holds 4 consecutive n of one row m and stores them together.
//
// 16-bit operands go from memory to LDS directly (buffer_load_dwordx4 ... lds) where rows are aligned to 16
// bytes, else through registers.  fp32 operands are split exactly into three bf16 parts of 8 bits,
// x = x1 + x2 + x3: x1 is x cut off (rounded, the largest numbers would become infinities), x2 the remainder rounded
// to nearest, and what that leaves has 8 bits.  With |x2| <= 2^-7 |x| and |x3| <= 2^-16 |x| the six products of
// order >= 2^-16 are summed in fp32 on the bf16 matrix cores; x2 w3 + x3 w2 + x3 w3 is left out, 2^-22 |x||w| at most
// and of either sign (with x2 cut off, too, it was twice that and always the product's).  Six bf16 products at 2.5 PFLOP/s
// are 0.42 PFLOP/s, against 0.157 of the fp32 matrix instructions.
//
// Measured (medians of 60 calls), [8192 x 4096] [8192 x 4096]^T bf16 with gelu and a residual: forward 540 us (425 the
// main loop, 1.29 PFLOP/s), dx 434, dw 459, dh 93; [53000 x 128] [3920 x 128]^T fp32: 387, 321 and 344 us.
#include "elements.hpp"

#include <math.h>

namespace smlvm {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef int i32x4 __attribute__((ext_vector_type(4)));
#define LDS_PTR(T) __attribute__((address_space(3))) T*

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3, kSigmoid = 4, kTanh = 5 };

// FAST (16-bit results): reciprocals and exponentials of the hardware's precision, and Phi(h) from a fit of
// log(erfc(z) e^(z^2) / t) by a polynomial in t = 1 / (1 + 0.3 z) on 0 <= z <= 9.5 (least squares, reweighted to an
// even error of 4.3e-7): gelu is off by 2e-7 at most, a twentieth of half a step of fp16 near 0.01, and
// costs 14 instructions where erff, both of whose branches a wave takes, costs 50 (the 8192 x 8192 forward
// with it spent 300 us of 820 in the epilogue).
template <bool FAST>
__device__ __forceinline__ float sigmoid_f(float h)
{
    if constexpr (FAST) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * h));
    // fp32: e^-h = 2^y (1 + ln2 d) with y + d = -h log2 e to 48 bits; off by 7 half steps at most (2 from v_exp, 2 from
    // v_rcp, one each from the sums and the product), in a third of the instructions of expf and a division
    // ([42803 x 16] [6336 x 16]^T with silu and a residual: 945 -> 800 us).  From -89 on 2^y is infinite and the result
    // 0: not 1 / (1 + e^88), which times -3e38 is -2 (the clamp keeps d finite).
    const float g = fminf(fmaxf(h, -104.0f), 104.0f), y = -1.44269504f * g;
    const float d = fmaf(-g, 1.44269504f, -y) + g * -1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(y) * fmaf(0.693147181f, d, 1.0f), s = __builtin_amdgcn_rcpf(1.0f + e);
    return h != h ? h : s;
}
// the normal distribution function
template <bool FAST>
__device__ __forceinline__ float phi_f(float h)
{
    if constexpr (FAST) {
        const float z = fabsf(h) * 0.70710678f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, z, 1.0f));
        float p = 0.485700458f;
        p = fmaf(p, t, -1.98586082f);
        p = fmaf(p, t, 2.91078472f);
        p = fmaf(p, t, -2.12544775f);
        p = fmaf(p, t, 1.27865398f);
        p = fmaf(p, t, 0.173279762f);
        p = fmaf(p, t, 1.04183877f);
        p = fmaf(p, t, -1.77894974f);
        const float half = 0.5f * t * __builtin_amdgcn_exp2f(fmaf(-z, z, p) * 1.44269504f);
        return h >= 0.0f ? 1.0f - half : half;
    } else {
        return 0.5f * erfcf(h * -0.70710678118654752f);   // (1 + erf has no digits left below -5)
    }
}

// act, and its slope, for 8 elements: one (uniform) branch for all, not one each ([42803 x 16] [6336 x 16]^T fp32 with
// silu and a residual 800 -> 469 us; 8192 x 8192 x 4096 bf16 with gelu and a residual 548 -> 507)
template <bool FAST>
__device__ __forceinline__ void act_all(int act, float (&h)[8])
{
    auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = f(h[j]);
    };
    switch (act) {
        case kRelu: each([](float h) { return h > 0.0f ? h : (h != h ? h : 0.0f); }); break;
        case kGelu: each([](float h) { return h * phi_f<FAST>(h); }); break;
        case kSilu: each([](float h) { return h * sigmoid_f<FAST>(h); }); break;
        case kSigmoid: each([](float h) { return sigmoid_f<FAST>(h); }); break;
        case kTanh: each([](float h) { return tanhf(h); }); break;
        default: break;
    }
}
// y *= act'(h)
template <bool FAST>
__device__ __forceinline__ void slope_all(int act, const float (&h)[8], float (&y)[8])
{
    auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= f(h[j]);
    };
    switch (act) {
        case kRelu: each([](float h) { return h > 0.0f ? 1.0f : 0.0f; }); break;
        case kGelu: each([](float h) {
            const float e = FAST ? __builtin_amdgcn_exp2f(-0.72134752f * h * h) : expf(-0.5f * h * h);
            return fmaf(h * 0.39894228040143268f, e, phi_f<FAST>(h));
        }); break;
        case kSilu: each([](float h) { const float s = sigmoid_f<FAST>(h); return s * (1.0f + h * (1.0f - s)); }); break;
        case kSigmoid: each([](float h) { const float s = sigmoid_f<FAST>(h); return s * (1.0f - s); }); break;
        case kTanh: each([](float h) { const float t = tanhf(h); return 1.0f - t * t; }); break;
        default: break;
    }
}

struct GemmArgs {
    const void *a, *b;
    int64_t lda, ldb;             // elements between rows (k rows of a column operand)
    int64_t M, N, K;
    int64_t k_split;              // k range of one part, a multiple of the k tile
    void* out;                    // [M][N]
    const void *bias, *res;       // nullable; res [M][N] with row stride ldr
    int64_t ldr;
    void* pre;                    // nullable: act's argument [M][N]
    float* part;                  // not null: fp32 partial sums [splits][M][N] instead of out
    float* colsum_part;           // not null (column a, split): fp32 sums over k of A(m, k), [splits][M]
    void* colsum;                 // not null (column a): sums over k of A(m, k), [M]
    int act;
    int tiles_m, tiles_n;
};

// ----------------------------------------------------------------------------------- epilogue
// 8 consecutive elements, aligned to the element only; `have` of them exist
template <class T>
__device__ __forceinline__ void load8(const T* p, int have, float (&x)[8])
{
    if (have == 8) {
        constexpr int P = 16 / (int)sizeof(T);
        T t[8];
#pragma unroll
        for (int i = 0; i < 8 / P; ++i) {
            const u32x4 raw = reinterpret_cast<const u32x4_any*>(p)[i];
            __builtin_memcpy(&t[i * P], &raw, 16);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j < have ? (float)p[j] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int have, const float (&x)[8])
{
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = (T)x[j];
    if (have == 8) {
        constexpr int P = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / P; ++i) {
            u32x4 raw;
            __builtin_memcpy(&raw, &t[i * P], 16);
            reinterpret_cast<u32x4_any*>(p)[i] = raw;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < have) p[j] = t[j];
    }
}

// act's argument for the backward: fp32, next to bf16 tensors fp16.  The slope is taken from it, and its rounding must
// not add to that of dh and of the gradient itself (two roundings, 1.41 times one): with bf16 the gradients of bf16
// tensors were 1.6 times one rounding off, with fp16 those of fp16 tensors 1.52 times; with 3 bits more (fp16
// next to bf16) and with fp32 1.42.  Beyond fp16's range every activation's slope is constant; below it every one
// is continuous but relu's, whose positive arguments stay positive.
// Of relu's argument only the sign is read: fp16 next to fp16, too.
template <class T>
__device__ __forceinline__ void store_pre(void* pre, int64_t at, int have, const float (&x)[8], int act)
{
    const bool relu = act == kRelu;
    if (sizeof(T) == 4 || (KindOf<T>::value == SMLVM_F16 && !relu)) {
        store8(static_cast<float*>(pre) + at, have, x);
        return;
    }
    float h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = x[j] != x[j] ? x[j] : fminf(fmaxf(x[j], -65504.0f), 65504.0f);
    if (relu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = h[j] > 0.0f ? fmaxf(h[j], 0x1p-24f) : h[j];
    }
    store8(static_cast<f16_t*>(pre) + at, have, h);
}

// 8 consecutive n of row m: bias, activation, residual, stores
template <class T>
__device__ __forceinline__ void finish8(const GemmArgs& g, int64_t m, int64_t n, int have, float (&x)[8], const float (&b)[8], const float (&r)[8])
{
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += b[j];
    }
    if (g.pre) store_pre<T>(g.pre, m * g.N + n, have, x, g.act);
    act_all<sizeof(T) == 2>(g.act, x);
    if (g.res) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += r[j];
    }
    store8(static_cast<T*>(g.out) + m * g.N + n, have, x);
}
template <class T>
__device__ __forceinline__ void finish8(const GemmArgs& g, int64_t m, int64_t n, float (&x)[8], int most = 8)
{
    const int have = g.N - n < most ? (int)(g.N - n) : most;
    float r[8], b[8];
    if (g.res) load8(static_cast<const T*>(g.res) + m * g.ldr + n, have, r);
    if (g.bias) load8(static_cast<const T*>(g.bias) + n, have, b);
    finish8<T>(g, m, n, have, x, b, r);
}

// ------------------------------------------------------------------------------------- staging
// A tile of ROWS m (n) by BK k.  Row operand in LDS: [ROWS][BK] 16-bit elements, the 16-byte slots of a row
// exchanged by slot ^ f(row); column operand: [BK][ROWS], the 32-byte chunks of a k row exchanged by
// chunk ^ f(k).  The fs put the addresses that one LDS cycle serves on different banks: for 16-byte reads lanes 0-3,
// 12-15, 20-27 (and the like), for the transposing 8-byte ones 32 neighbours, that is k rows 0-3 and 8-11.
// (With f = row / 4 and f = k & 7 a fifth of the LDS cycles of dw's kernel were conflicts.)
template <int ROWS, int BK, bool COL>
struct Tile {
    static constexpr int kBytes = ROWS * BK * 2;
    static constexpr int kSlots = kBytes / 16;
    static constexpr int kPerRow = (COL ? ROWS : BK) / 8;               // slots per stored row
    static constexpr int kMask = COL ? (ROWS / 16 < 8 ? ROWS / 16 : 8) - 1 : kPerRow - 1;
    static_assert(BK == 32 || BK == 64, "swizzles below");

    __device__ __forceinline__ static int swizzle(int row)
    {
        if constexpr (COL) {
            return kMask == 7 ? (row & 3) | ((row >> 1) & 4) : ((row >> 1) & 1) | ((row >> 2) & 2);
        } else if constexpr (kPerRow == 8) {
            return (row >> 1) & 7;
        } else {
            const int r = (row >> 2) & 3;
            return (((r ^ (r >> 1)) & 1) << 1) | (r >> 1);
        }
    }
    // 16-byte slot -> (stored row, first element in it) of the source
    __device__ __forceinline__ static void source(int slot, int& row, int& at)
    {
        row = slot / kPerRow;
        const int s = slot % kPerRow;
        if constexpr (COL) at = (((s >> 1) ^ swizzle(row)) << 4) + ((s & 1) << 3);
        else at = (s ^ swizzle(row)) << 3;
    }
    // lane's 8 k of row `base + lane % 16`, k step kk (of 32): byte offset (row operand)
    __device__ __forceinline__ static int row_at(int base, int kk, int lane)
    {
        const int row = base + (lane & 15), s = kk * 4 + (lane >> 4);
        return row * (BK * 2) + ((s ^ swizzle(row)) << 4);
    }
    // column operand: p-th (of two) transposing reads
    __device__ __forceinline__ static int col_at(int base, int kk, int p, int lane)
    {
        const int k = kk * 32 + ((lane >> 4) << 3) + p * 4 + ((lane & 15) >> 2);
        return k * (ROWS * 2) + (((base >> 4) ^ swizzle(k)) << 5) + ((lane & 3) << 3);
    }
    __device__ __forceinline__ static s16x8 fragment(const char* tile, int base, int kk, int lane)
    {
        if constexpr (COL) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(tile + col_at(base, kk, 0, lane)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(tile + col_at(base, kk, 1, lane)));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const s16x8*>(tile + row_at(base, kk, lane));
        }
    }
};

template <class T>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c)
{
    if constexpr (sizeof(T) == 2 && KindOf<T>::value == SMLVM_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16 bytes per lane from memory to LDS, in flight until the next wait_loads().  The lane's LDS address is
// `lds` + 16 * lane; offsets beyond the resource's range leave zeros.
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t offset, uint32_t lds)
{
    // (4 idle states: the resource may just have been written by a vector instruction; m0 has no other use
    // in these kernels)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(offset), "s"(rsrc), "s"(lds) : "memory");
}
__device__ __forceinline__ void wait_loads_and_sync()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
constexpr uint32_t kOutside = 0x80000000u;                              // = the resource's range
__device__ __forceinline__ i32x4 resource(const void* p)
{
    const uint64_t a = (uint64_t)p;
    i32x4 r = {__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xFFFF),
               (int)kOutside, 0x00020000};
    return r;
}

// Direct staging of one operand: each thread owns kSlots / THREADS slots, whose offsets into the source
// (relative to the tile's first row and the current k) never change.
template <int ROWS, int BK, bool COL, int THREADS>
struct Direct {
    using Tl = Tile<ROWS, BK, COL>;
    static constexpr int kEach = Tl::kSlots / THREADS;
    static_assert(Tl::kSlots % THREADS == 0, "whole slots per thread");
    uint32_t offset[kEach];
    int k_of[kEach];                                                    // k within the tile (slots are all in or all out)

    __device__ __forceinline__ void init(int64_t ld, int64_t first, int64_t extent)
    {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            int row, at;
            Tl::source(i * THREADS + threadIdx.x, row, at);
            k_of[i] = COL ? row : at;
            const int64_t m = first + (COL ? at : row);
            offset[i] = m < extent ? (uint32_t)((row * ld + at) * 2) : kOutside;
        }
    }
    // `base`: the tile's first row at the current k
    __device__ __forceinline__ void issue(const char* base, int64_t k_left, uint32_t lds) const
    {
        const i32x4 rsrc = resource(base);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t wave = __builtin_amdgcn_readfirstlane((i * THREADS + (threadIdx.x & ~63)) * 16);
            load_to_lds(rsrc, k_of[i] < k_left ? offset[i] : kOutside, lds + wave);
        }
    }
};

// Staging through registers: fp32 (split into three planes on the way) and 16-bit operands whose rows are
// not aligned.
template <class T, int ROWS, int BK, bool COL, int THREADS>
struct Through {
    using Tl = Tile<ROWS, BK, COL>;
    static constexpr int kEach = Tl::kSlots / THREADS;
    static constexpr int kVecs = (int)sizeof(T) / 2;                    // 16-byte loads per 8 elements
    static_assert(Tl::kSlots % THREADS == 0, "whole slots per thread");
    u32x4 held[kEach][kVecs];
    const T* from[kEach];                                               // the slot's elements at the current k
    int64_t ld, step;

    __device__ __forceinline__ void init(const T* src, int64_t ld_, int64_t first, int64_t k0)
    {
        ld = ld_;
        step = COL ? BK * ld : BK;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            int row, at;
            Tl::source(i * THREADS + threadIdx.x, row, at);
            from[i] = COL ? src + (k0 + row) * ld + first + at : src + (first + row) * ld + k0 + at;
        }
    }
    // `rows`: what is left of the matrix' m (n), `k_left` of this part's k, `k_all` of the matrix'; then on to the
    // next k tile.  At an edge a slot that ends behind its row is read whole where that much of the matrix
    // follows (the elements too many are of an m nobody stores, or a k that is cleared here), element by
    // element at its end.
    __device__ __forceinline__ void load(int64_t rows, int64_t k_left, int64_t k_all)
    {
        if (rows >= ROWS && k_left >= BK) {                             // (uniform)
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
#pragma unroll
                for (int v = 0; v < kVecs; ++v) held[i][v] = reinterpret_cast<const u32x4_any*>(from[i])[v];
                from[i] += step;
            }
            return;
        }
        const int r_end = (int)(COL ? (k_left < BK ? k_left : BK) : (rows < ROWS ? rows : ROWS));
        const int c_end = (int)(COL ? (rows < ROWS ? rows : ROWS) : (k_left < BK ? k_left : BK));
        const int64_t r_all = COL ? k_all : rows, c_all = COL ? rows : k_all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            int row, at;
            Tl::source(i * THREADS + threadIdx.x, row, at);
            const bool in = row < r_end && at < c_end;
            const bool whole = at + 8 <= c_end || at + 8 <= (r_all - 1 - row) * ld + c_all;
#pragma unroll
            for (int v = 0; v < kVecs; ++v) held[i][v] = u32x4{0u, 0u, 0u, 0u};
            if (in && whole) {
#pragma unroll
                for (int v = 0; v < kVecs; ++v) held[i][v] = reinterpret_cast<const u32x4_any*>(from[i])[v];
            }
            if (in && !whole) {
                T t[8] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) if (at + j < c_end) t[j] = from[i][j];
                __builtin_memcpy(held[i], t, 8 * sizeof(T));
            }
            from[i] += step;
        }
        if (!COL && k_left < BK) {                                      // (uniform) clear the k behind the last one
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                int row, at;
                Tl::source(i * THREADS + threadIdx.x, row, at);
                const int have = c_end - at;
#pragma unroll
                for (int v = 0; v < kVecs; ++v)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = (v * 4 + j) * 4 / (int)sizeof(T);  // the word's first element
                        if constexpr (sizeof(T) == 4) held[i][v][j] = e < have ? held[i][v][j] : 0u;
                        else held[i][v][j] &= e + 1 < have ? 0xFFFFFFFFu : e < have ? 0xFFFFu : 0u;
                    }
            }
        }
    }
    // planes: 1 (16-bit) or 3 (fp32), each a whole tile
    __device__ __forceinline__ void store(char* tile) const
    {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            char* const to = tile + (i * THREADS + threadIdx.x) * 16;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<u32x4*>(to) = held[i][0];
            } else {
                u32x4 plane[3];
#pragma unroll
                for (int j = 0; j < 4; ++j) {                            // two elements -> one word of each plane
                    float x[2];
                    const uint32_t raw[2] = {held[i][j >> 1][(j & 1) * 2], held[i][j >> 1][(j & 1) * 2 + 1]};
                    plane[0][j] = __builtin_amdgcn_perm(raw[1], raw[0], 0x07060302);   // high halves
#pragma unroll
                    for (int e = 0; e < 2; ++e) x[e] = __builtin_bit_cast(float, raw[e]) - __builtin_bit_cast(float, raw[e] & 0xFFFF0000u);
                    plane[1][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[0], x[1]}), bf16x2));
                    x[0] -= __builtin_bit_cast(float, plane[1][j] << 16);
                    x[1] -= __builtin_bit_cast(float, plane[1][j] & 0xFFFF0000u);
                    plane[2][j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[1]), __builtin_bit_cast(uint32_t, x[0]), 0x07060302);
                }
#pragma unroll
                for (int q = 0; q < 3; ++q) *reinterpret_cast<u32x4*>(to + q * Tl::kBytes) = plane[q];
            }
        }
    }
};

// ------------------------------------------------------------------------------------ the kernel
// BM x BN tile, WM x WN waves, DIRECT: 16-bit aligned operands.  Through registers one LDS buffer does: the next
// tile waits in registers, and two or three workgroups per CU fill each other's gaps (two buffers of the fp32
// planes would leave room for one).
template <class T, int BM, int BN, bool DIRECT> constexpr int kBuffers = DIRECT || (sizeof(T) == 4 && BM == 256) ? 2 : 1;
template <class T, int BM, int BN, bool DIRECT>
constexpr int kLdsBytes = kBuffers<T, BM, BN, DIRECT> * (BM + BN) * (sizeof(T) == 4 ? 3 * 32 : 64) * 2;

// tile `id` of part `part_z`
template <class T, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, bool DIRECT>
__device__ __forceinline__ void gemm_body(const GemmArgs& g, int id, int part_z, char* lds)
{
    constexpr int THREADS = WM * WN * 64;
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int BK = SPLIT ? 32 : 64;
    constexpr int PLANES = SPLIT ? 3 : 1;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;                 // 16 x 16 tiles per wave
    using TA = Tile<BM, BK, ACOL>;
    using TB = Tile<BN, BK, BCOL>;
    constexpr int STAGE = PLANES * (TA::kBytes + TB::kBytes);
    constexpr int BUFFERS = kBuffers<T, BM, BN, DIRECT>;
    static_assert(kLdsBytes<T, BM, BN, DIRECT> == BUFFERS * STAGE, "LDS");

    // (wave in a scalar register: matrix instructions ignore the exec mask, so what skips one has to be a
    // scalar branch)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go round the 8 XCDs: give each XCD, with its own L2, one stretch of tiles, walked in
    // groups of 8 row tiles so that its neighbours share operands.
    const int tiles = g.tiles_m * g.tiles_n;
    {
        const int per = tiles / 8, rest = tiles % 8, xcd = id % 8, at = id / 8;
        id = xcd * per + (xcd < rest ? xcd : rest) + at;
    }
    const int group = id / (8 * g.tiles_n), first_m = group * 8;
    const int rows_here = g.tiles_m - first_m < 8 ? g.tiles_m - first_m : 8;
    const int in_group = id - group * 8 * g.tiles_n;
    const int64_t m0 = (int64_t)(first_m + in_group % rows_here) * BM;
    const int64_t n0 = (int64_t)(in_group / rows_here) * BN;
    const int64_t k_begin = (int64_t)part_z * g.k_split;
    const int64_t k_end = g.K < k_begin + g.k_split ? g.K : k_begin + g.k_split;
    const int mw = (wave / WN) * (BM / WM), nw = (wave % WN) * (BN / WN);
    const bool colsum = ACOL && g.colsum && n0 == 0;
    constexpr int FS = ACOL ? FM / WN : 1;                              // a wave's share of its rows' column sums

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 sums[FS];
#pragma unroll
    for (int i = 0; i < FS; ++i) sums[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr short kOne = KindOf<T>::value == SMLVM_F16 ? 0x3C00 : 0x3F80;
    const s16x8 ones = {kOne, kOne, kOne, kOne, kOne, kOne, kOne, kOne};

    auto compute = [&](const char* stage) {
        const char* const ta = stage;
        const char* const tb = stage + PLANES * TA::kBytes;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            if constexpr (FM * FN >= 32 && ACOL) __builtin_amdgcn_sched_barrier(0);   // (one step's operands at a time: registers)
            s16x8 af[PLANES][FM], bf[PLANES][FN];
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
#pragma unroll
                for (int j = 0; j < FN; ++j) bf[q][j] = TB::fragment(tb + q * TB::kBytes, nw + j * 16, kk, lane);
#pragma unroll
                for (int i = 0; i < FM; ++i) af[q][i] = TA::fragment(ta + q * TA::kBytes, mw + i * 16, kk, lane);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    if constexpr (SPLIT) {                              // smallest terms first
                        acc[i][j] = mfma<T>(bf[2][j], af[0][i], acc[i][j]);
                        acc[i][j] = mfma<T>(bf[0][j], af[2][i], acc[i][j]);
                        acc[i][j] = mfma<T>(bf[1][j], af[1][i], acc[i][j]);
                        acc[i][j] = mfma<T>(bf[1][j], af[0][i], acc[i][j]);
                        acc[i][j] = mfma<T>(bf[0][j], af[1][i], acc[i][j]);
                    }
                    acc[i][j] = mfma<T>(bf[0][j], af[0][i], acc[i][j]);
                }
            if constexpr (ACOL) {
                if (colsum) {
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        if (i / FS != wave % WN) continue;               // (uniform)
#pragma unroll
                        for (int q = PLANES - 1; q >= 0; --q) sums[i % FS] = mfma<T>(ones, af[q][i], sums[i % FS]);
                    }
                }
            }
        }
    };

    // The order wanted of a step of the largest 16-bit tiles: the first 32 k's LDS reads, then the second's among the
    // first matrix instructions (8192 x 8192 x 4096: 455 -> 425 us, dx 443 -> 418; dw, whose reads are twice as
    // many, has no registers left for it).
    auto order = [&] {
        if constexpr (DIRECT && FM * FN >= 32 && !ACOL) {
            constexpr int READS = FM + FN * (BCOL ? 2 : 1);
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, FM * FN / READS, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * FM * FN - FM * FN / READS * READS, 0);
        }
    };
    const T* const a = static_cast<const T*>(g.a);
    const T* const b = static_cast<const T*>(g.b);
    const int64_t steps = k_end > k_begin ? (k_end - k_begin + BK - 1) / BK : 0;
    if constexpr (DIRECT) {
        static_assert(!SPLIT, "fp32 goes through registers");
        Direct<BM, BK, ACOL, THREADS> sa;
        Direct<BN, BK, BCOL, THREADS> sb;
        sa.init(g.lda, m0, g.M);
        sb.init(g.ldb, n0, g.N);
        const char* pa = reinterpret_cast<const char*>(ACOL ? a + k_begin * g.lda + m0 : a + m0 * g.lda + k_begin);
        const char* pb = reinterpret_cast<const char*>(BCOL ? b + k_begin * g.ldb + n0 : b + n0 * g.ldb + k_begin);
        const int64_t ka = (ACOL ? g.lda : 1) * (BK * 2), kb = (BCOL ? g.ldb : 1) * (BK * 2);
        const uint32_t base = (uint32_t)(uintptr_t)(LDS_PTR(char))lds;
        auto issue = [&](int64_t step, int buf) {
            const int64_t left = k_end - k_begin - step * BK;
            sa.issue(pa + step * ka, left, base + buf * STAGE);
            sb.issue(pb + step * kb, left, base + buf * STAGE + TA::kBytes);
        };
        if (steps > 0) issue(0, 0);
        for (int64_t s = 0; s < steps; ++s) {
            // (this tile has arrived, and everybody is done with the buffer that is filled next)
            wait_loads_and_sync();
            if (s + 1 < steps) issue(s + 1, (int)((s + 1) & 1));
            compute(lds + (s & 1) * STAGE);
            order();
        }
    } else {
        Through<T, BM, BK, ACOL, THREADS> sa;
        Through<T, BN, BK, BCOL, THREADS> sb;
        sa.init(a, g.lda, m0, k_begin);
        sb.init(b, g.ldb, n0, k_begin);
        if (steps > 0) {
            sa.load(g.M - m0, k_end - k_begin, g.K - k_begin);
            sb.load(g.N - n0, k_end - k_begin, g.K - k_begin);
        }
        auto next = [&](int64_t step) {
            const int64_t left = k_end - k_begin - step * BK, all = g.K - k_begin - step * BK;
            sa.load(g.M - m0, left, all);
            sb.load(g.N - n0, left, all);
        };
        auto put = [&](char* stage) {
            sa.store(stage);
            sb.store(stage + PLANES * TA::kBytes);
        };
        if constexpr (BUFFERS == 2) {
            // The next tile is split and written while this one is multiplied: one barrier per step, and the
            // vector work between the matrix instructions of the same wave (4096^3: 642 us as the compiler
            // orders it, 592 as asked for below: 232 TFLOP/s, 1.39 PFLOP/s of bf16 products).
            if (steps > 0) put(lds);
            if (steps > 1) next(1);
            for (int64_t s = 0; s < steps; ++s) {
                __syncthreads();
                compute(lds + (s & 1) * STAGE);
                put(lds + ((s + 1) & 1) * STAGE);                        // (after the last step: what nobody reads)
                // the order wanted: the step's LDS reads, then 4 matrix and 6 vector instructions in turn
                __builtin_amdgcn_sched_group_barrier(0x100, PLANES * (FM * (ACOL ? 2 : 1) + FN * (BCOL ? 2 : 1)), 0);
#pragma unroll
                for (int i = 0; i < FM * FN * 6 / 4; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                    if (i % 2 == 1) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
                }
                if (s + 2 < steps) next(s + 2);
            }
        } else {
            for (int64_t s = 0; s < steps; ++s) {
                __syncthreads();                                         // (the last tile has been read)
                put(lds);
                __syncthreads();
                if (s + 1 < steps) next(s + 1);
                compute(lds);
            }
        }
    }

    // 16 rows at a time through the wave's own part of the LDS: a lane holds 4 n of one row, and stores 8 of
    // another, so that a row's stores fill whole cache lines.  (Rows 16 bytes apart in bank: no conflicts.)
    constexpr int COLS = BN / WN, PITCH = COLS + 4, PER_ROW = COLS / 8, V = 16 * PER_ROW / 64;
    static_assert(WM * WN * 16 * PITCH * 4 <= BUFFERS * STAGE, "epilogue tile");
    static_assert(64 % PER_ROW == 0, "a lane's columns stay the same");
    __syncthreads();
    float* const own = reinterpret_cast<float*>(lds) + wave * (16 * PITCH);
    const int64_t n = n0 + nw + lane % PER_ROW * 8, m_first = m0 + mw + lane / PER_ROW;
    const int have = n >= g.N ? 0 : g.N - n < 8 ? (int)(g.N - n) : 8;
    // the bias is loaded once, the residual 16 rows ahead: a load's latency in front of every store is what it cost
    float bias[8], ahead[V][8];
    const bool finishes = !g.part;
    if (finishes && g.bias && have) load8(static_cast<const T*>(g.bias) + n, have, bias);
    auto fetch = [&](int i) {
        if (!finishes || !g.res || !have) return;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int64_t m = m_first + i * 16 + v * (64 / PER_ROW);
            if (m < g.M) load8(static_cast<const T*>(g.res) + m * g.ldr + n, have, ahead[v]);
        }
    };
    fetch(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        if constexpr (ACOL) {
            const int64_t m = m0 + mw + i * 16 + lane;
            if (colsum && lane < 16 && m < g.M && i / FS == wave % WN) {
                if (g.colsum_part) g.colsum_part[(int64_t)part_z * g.M + m] = sums[i % FS].x;
                else static_cast<T*>(g.colsum)[m] = (T)sums[i % FS].x;
            }
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
            *reinterpret_cast<f32x4*>(own + (lane & 15) * PITCH + j * 16 + ((lane >> 4) << 2)) = acc[i][j];
        wave_lds_sync();
        float x[V][8], r[V][8];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            load_vec<float, 8>(own + (v * (64 / PER_ROW) + lane / PER_ROW) * PITCH + lane % PER_ROW * 8, x[v]);
#pragma unroll
            for (int j = 0; j < 8; ++j) r[v][j] = ahead[v][j];
        }
        if (i + 1 < FM) fetch(i + 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int64_t m = m_first + i * 16 + v * (64 / PER_ROW);
            if (m < g.M && have) {
                if (g.part) store8(g.part + ((int64_t)part_z * g.M + m) * g.N + n, have, x[v]);
                else finish8<T>(g, m, n, have, x[v], bias, r[v]);
            }
        }
        wave_lds_sync();
    }
}

template <class T, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(const GemmArgs g)
{
    __shared__ __attribute__((aligned(16))) char lds[kLdsBytes<T, BM, BN, DIRECT>];
    gemm_body<T, ACOL, BCOL, BM, BN, WM, WN, DIRECT>(g, blockIdx.x, blockIdx.z, lds);
}

// A layer's two backward products in one launch, where neither fills the card by itself: [1001 x 777] with
// [777 x 333] and [333 x 1001], fp16, 27 us one after the other.
template <class T, bool DIRECT>
__global__ __launch_bounds__(256) void pair_kernel(const GemmArgs dx, const GemmArgs dw, int blocks_dx)
{
    __shared__ __attribute__((aligned(16))) char lds[kLdsBytes<T, 64, 64, DIRECT>];
    const int id = blockIdx.x;
    if (id < blocks_dx) {
        const int tiles = dx.tiles_m * dx.tiles_n;
        gemm_body<T, false, true, 64, 64, 2, 2, DIRECT>(dx, id % tiles, id / tiles, lds);
    } else {
        const int tiles = dw.tiles_m * dw.tiles_n;
        gemm_body<T, true, true, 64, 64, 2, 2, DIRECT>(dw, (id - blocks_dx) % tiles, (id - blocks_dx) / tiles, lds);
    }
}

// Few rows (M <= kFewRows): bound by reading w once.  A wave owns two rows of w, its lanes go along k 16 bytes at a
// time, x comes out of the caches; the sums are joined across the lanes at the end.  One launch, where the tiled
// kernel needs a split over k and a join: [1 x 4096] [4096 x 4096]^T bf16 takes 8.6 us against 10.7.
constexpr int kFewRows = 4;
template <class T, int MR>
__global__ __launch_bounds__(256) void few_rows_kernel(const GemmArgs g)
{
    constexpr int P = 16 / (int)sizeof(T), NW = 2, U = MR <= 2 ? 4 : 2;
    const int lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * NW;
    if (n0 >= g.N) return;
    const T* const x = static_cast<const T*>(g.a);
    const T* w[NW];
#pragma unroll
    for (int c = 0; c < NW; ++c) w[c] = static_cast<const T*>(g.b) + (n0 + c < g.N ? n0 + c : n0) * g.ldb;
    float acc[MR][NW] = {};
    const int64_t whole = g.K / P * P;
    int64_t k = (int64_t)lane * P;
    auto step = [&](const u32x4 (&wv)[NW], int64_t at) {
        T wt[NW][P];
#pragma unroll
        for (int c = 0; c < NW; ++c) __builtin_memcpy(wt[c], &wv[c], 16);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const u32x4 xv = *reinterpret_cast<const u32x4_any*>(x + m * g.lda + at);
            T xt[P];
            __builtin_memcpy(xt, &xv, 16);
#pragma unroll
            for (int c = 0; c < NW; ++c)
#pragma unroll
                for (int j = 0; j < P; ++j) acc[m][c] = fmaf((float)xt[j], (float)wt[c][j], acc[m][c]);
        }
    };
    for (; k + (U - 1) * 64 * P < whole; k += U * 64 * P) {
        u32x4 wv[U][NW];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < NW; ++c) wv[u][c] = *reinterpret_cast<const u32x4_any*>(w[c] + k + u * 64 * P);
#pragma unroll
        for (int u = 0; u < U; ++u) step(wv[u], k + u * 64 * P);
    }
    for (; k < whole; k += 64 * P) {
        u32x4 wv[NW];
#pragma unroll
        for (int c = 0; c < NW; ++c) wv[c] = *reinterpret_cast<const u32x4_any*>(w[c] + k);
        step(wv, k);
    }
    if (whole + lane < g.K) {
        const int64_t at = whole + lane;
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int c = 0; c < NW; ++c) acc[m][c] = fmaf((float)x[m * g.lda + at], (float)w[c][at], acc[m][c]);
    }
    float mine = 0.0f;                                                   // lane m * NW + c keeps sum (m, c)
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int c = 0; c < NW; ++c) {
            const float sum = group_reduce<64>(acc[m][c], OpSum{});
            if (lane == m * NW + c) mine = sum;
        }
    const int64_t n = n0 + lane % NW;
    if (lane < MR * NW && n < g.N) {
        float one[8] = {mine};
        finish8<T>(g, lane / NW, n, one, 1);
    }
}

// Joins the partial sums of a split product, in order, and runs the epilogue; the workgroups behind the
// first `blocks` join the column sums.
struct Join {
    int splits, blocks;               // of the partial products
    const float* sums;                // partial column sums [parts][n], joined by sum_blocks workgroups
    int parts, sum_blocks;
    int64_t n;
    void* sum_out;
};
template <class T>
__device__ __forceinline__ void join_body(const GemmArgs& g, const Join& p, int id)
{
    const int splits = p.splits, blocks = p.blocks;
    if (id >= blocks) {                                                  // 64 sums, every fourth part to a wave
        __shared__ float quarter[4][64];
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const int64_t m = (int64_t)(id - blocks) * 64 + lane;
        float s = 0.0f;
        if (m < p.n) {
#pragma unroll 8
            for (int z = wave; z < p.parts; z += 4) s += p.sums[(int64_t)z * p.n + m];
        }
        quarter[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && m < p.n)
            static_cast<T*>(p.sum_out)[m] = (T)((quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]));
        return;
    }
    const int64_t per_row = (g.N + 7) / 8, total = g.M * per_row;
    for (int64_t v = (int64_t)id * 256 + threadIdx.x; v < total; v += (int64_t)blocks * 256) {
        const int64_t m = v / per_row, n = (v - m * per_row) * 8;
        const int have = g.N - n < 8 ? (int)(g.N - n) : 8;
        float x[8] = {};
        for (int z = 0; z < splits; ++z) {
            float y[8];
            load8<float>(g.part + ((int64_t)z * g.M + m) * g.N + n, have, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] += y[j];
        }
        finish8<T>(g, m, n, x);
    }
}

// one product's, and behind its workgroups another's
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const GemmArgs g, const Join p, const GemmArgs g2, const Join p2)
{
    const int id = blockIdx.x, first = p.blocks + p.sum_blocks;
    if (id < first) join_body<T>(g, p, id);
    else join_body<T>(g2, p2, id - first);
}

template <bool V> struct Flag { static constexpr bool value = V; };

// dh = dy act'(h), H the type h is kept in; relu may be given y in the place of h (the sign is the same).  The column
// sums db come from here, before dh is rounded: sums of rounded values are one rounding further off.  A workgroup owns
// 8 * groups columns (groups a power of two) of `rows` rows, 256 / groups rows at a time; sums [gridDim.y][N] are
// joined in order later.
template <class T, class H>
__global__ __launch_bounds__(256) void act_bwd_kernel(const T* __restrict__ dy, const H* __restrict__ h, T* __restrict__ dh,
                                                      int64_t M, int64_t N, int act, int groups, int64_t rows,
                                                      float* __restrict__ sums)
{
    __shared__ float shared[256 * 8];
    const int tx = threadIdx.x & (groups - 1), ty = threadIdx.x / groups, step = 256 / groups;
    const int64_t n = ((int64_t)blockIdx.x * groups + tx) * 8;
    const int have = n >= N ? 0 : N - n < 8 ? (int)(N - n) : 8;
    const int64_t last = (int64_t)(blockIdx.y + 1) * rows < M ? (int64_t)(blockIdx.y + 1) * rows : M;
    float total[8] = {};
    const int64_t end = M * N, first = (int64_t)blockIdx.y * rows + ty;
    auto walk = [&](auto even) {                                         // even: N is a multiple of 8
        constexpr bool EVEN = decltype(even)::value;
        // (the elements that a row's last lane reads too many are the next row's; the last row has none behind it)
        auto fetch = [&](int64_t at, float (&x)[8], float (&y)[8]) {
            const int width = EVEN || at + 8 <= end ? 8 : have;
            load8(h + at, width, x);
            load8(dy + at, width, y);
        };
        auto one = [&](float (&y)[8], const float (&x)[8], int64_t at) {
            slope_all<sizeof(T) == 2>(act, x, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) total[j] += y[j];
            store8(dh + at, EVEN ? 8 : have, y);
        };
        constexpr int U = 4;                                             // rows in flight
        int64_t m = first;
        for (; m + (U - 1) * step < last; m += U * step) {
            float x[U][8], y[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) fetch((m + u * step) * N + n, x[u], y[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) one(y[u], x[u], (m + u * step) * N + n);
        }
        for (; m < last; m += step) {
            float x[8], y[8];
            fetch(m * N + n, x, y);
            one(y, x, m * N + n);
        }
    };
    if (have) {
        if (N % 8 == 0) walk(Flag<true>{});
        else walk(Flag<false>{});
    }
    if (!sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) shared[threadIdx.x * 8 + j] = total[j];
    __syncthreads();
    if (ty == 0 && have) {
        for (int t = 1; t < step; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j) total[j] += shared[(t * groups + tx) * 8 + j];
        store8(sums + (int64_t)blockIdx.y * N + n, have, total);
    }
}

// -------------------------------------------------------------------------------------- host side
struct Plan { int bm, bn, splits; int64_t k_split; };

// Tile and split of k by the estimated time of each combination.  A workgroup costs `fixed` us plus, per k
// tile, its own latency or its share of the CU, whichever is more; a split adds the join's launch and
// its traffic.  The numbers are fits to products timed alone (us): 2048^3 bf16 with 64 / 128 / 256 tiles
// 25.6 / 26.5 / 57.8; [53000 x 3920]^T [53000 x 128] fp32 with 64 tiles in 5 parts 499, with 128 tiles in 16
// parts 344; [200 x 4000] [4000 x 4000]^T fp32 with 64 tiles whole 134, in 4 parts 63, with 128 tiles in 8 parts 53;
// 4096^3 fp32 with 128 x 128 tiles 629, with 256 x 128 tiles 592; [1 x 4096] [4096 x 4096]^T bf16 with 64 tiles whole 31, in 8 parts 10.7.
static Plan plan(int kind, int64_t M, int64_t N, int64_t K, bool direct)
{
    struct Tile { int bm, bn, slots; double fixed, latency, share; };
    static const Tile kF32[] = {{256, 128, 1, 9.0, 2.2, 2.2}, {128, 128, 2, 5.0, 1.80, 1.14}, {64, 64, 4, 3.0, 0.95, 0.45}};
    static const Tile kDirect[] = {{256, 256, 1, 14.0, 1.75, 1.75}, {128, 128, 2, 5.0, 0.75, 0.60}, {64, 64, 5, 2.5, 0.42, 0.18}};
    static const Tile kThrough[] = {{128, 128, 2, 6.0, 1.50, 0.95}, {64, 64, 5, 3.0, 0.85, 0.27}};
    const Tile* const set = kind == SMLVM_F32 ? kF32 : direct ? kDirect : kThrough;
    const int sizes = kind == SMLVM_F32 || direct ? 3 : 2;
    const int64_t bk = kind == SMLVM_F32 ? 32 : 64, k_tiles = (K + bk - 1) / bk;
    Plan best = {64, 64, 1, bk};
    double least = 1e300;
    for (int i = 0; i < sizes; ++i) {
        const Tile& t = set[i];
        const double tiles_n = N > 0 ? (double)((N + t.bn - 1) / t.bn) : 1.0;     // (N = 0: column sums alone)
        const double tiles = (double)((M + t.bm - 1) / t.bm) * tiles_n;
        for (int splits = 1; splits <= 64; splits += splits < 4 ? 1 : splits / 2) {
            const int64_t per = k_tiles > 0 ? (k_tiles + splits - 1) / splits : 1;
            if (splits > 1 && per < 4) break;
            const double each_cu = ceil(tiles * splits / 256.0);
            const double at_once = each_cu < t.slots ? each_cu : t.slots;
            const double step = t.latency > at_once * t.share ? t.latency : at_once * t.share;
            double time = ceil(each_cu / at_once) * (t.fixed + (double)per * step);
            if (splits > 1) time += 6.0 + (double)splits * (double)M * (double)N * 8.0 / 4.0e6;
            if (time < least) {
                least = time;
                best.bm = t.bm;
                best.bn = t.bn;
                best.k_split = per * bk;
                best.splits = (int)(k_tiles > 0 ? (k_tiles + per - 1) / per : 1);
            }
        }
    }
    return best;
}

static bool direct_ok(int kind, const void* p, int64_t ld, int64_t contiguous)
{
    // (a tile's byte offsets stay below 2^31: up to 256 rows)
    return kind != SMLVM_F32 && aligned16(p) && ld % 8 == 0 && contiguous % 8 == 0 && ld < (1 << 20);
}

template <class T, bool ACOL, bool BCOL>
static void launch_gemm(const Plan& p, bool direct, const GemmArgs& g, hipStream_t stream)
{
    const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), 1, (unsigned)p.splits);
#define GEMM(BM, BN, WM, WN, DIRECT) \
    hipLaunchKernelGGL((gemm_kernel<T, ACOL, BCOL, BM, BN, WM, WN, DIRECT>), grid, dim3(WM * WN * 64), 0, stream, g)
    if constexpr (sizeof(T) == 2) {
        if (direct) {
            if (p.bm == 256) GEMM(256, 256, 2, 4, true);
            else if (p.bm == 128) GEMM(128, 128, 2, 2, true);
            else GEMM(64, 64, 2, 2, true);
            return;
        }
    }
    if constexpr (sizeof(T) == 4) {
        if (p.bm == 256) {
            GEMM(256, 128, 4, 2, false);
            return;
        }
    }
    if (p.bm == 128) GEMM(128, 128, 2, 2, false);
    else GEMM(64, 64, 2, 2, false);
#undef GEMM
}

template <class T>
static void launch_few_rows(const GemmArgs& g, hipStream_t stream)
{
    const dim3 grid((unsigned)((g.N + 7) / 8));
    switch (g.M) {
        case 1: hipLaunchKernelGGL((few_rows_kernel<T, 1>), grid, dim3(256), 0, stream, g); break;
        case 2: hipLaunchKernelGGL((few_rows_kernel<T, 2>), grid, dim3(256), 0, stream, g); break;
        case 3: hipLaunchKernelGGL((few_rows_kernel<T, 3>), grid, dim3(256), 0, stream, g); break;
        default: hipLaunchKernelGGL((few_rows_kernel<T, 4>), grid, dim3(256), 0, stream, g); break;
    }
}

// One product, planned: layout 0: rows x rows, 1: rows x columns, 2: columns x columns.
struct Job {
    GemmArgs g;
    Plan p;
    bool direct;
    int layout;
    Join sums;                                       // column sums that another kernel has left in parts
};

// Plans a product and takes what it needs of the workspace.
static int plan_job(Job& j, int kind, int layout, void* colsum, char*& ws, size_t& left)
{
    GemmArgs& g = j.g;
    j.layout = layout;
    j.direct = direct_ok(kind, g.a, g.lda, layout == 2 ? g.M : g.K) && direct_ok(kind, g.b, g.ldb, layout ? g.N : g.K);
    j.p = plan(kind, g.M, g.N, g.K, j.direct);
    if (!grid_fits((double)((g.M + j.p.bm - 1) / j.p.bm) * (double)((g.N + j.p.bn - 1) / j.p.bn),
                   j.p.bm == 256 ? 512 : 256)) return SMLVM_ERR_UNSUPPORTED;
    g.tiles_m = (int)((g.M + j.p.bm - 1) / j.p.bm);
    g.tiles_n = (int)((g.N + j.p.bn - 1) / j.p.bn);
    if (g.tiles_n == 0) g.tiles_n = 1;               // (column sums alone)
    g.k_split = j.p.k_split;
    g.colsum = colsum;
    if (j.p.splits > 1) {
        const size_t part = (size_t)j.p.splits * g.M * g.N, sums = colsum ? (size_t)j.p.splits * g.M : 0;
        const size_t need = (part + sums) * sizeof(float);
        if (!ws || left < need) return SMLVM_ERR_WORKSPACE;
        g.part = reinterpret_cast<float*>(ws);
        if (colsum) g.colsum_part = g.part + part;
        ws += need;
        left -= need;
    }
    return SMLVM_OK;
}

static Join join_of(const Job& j)
{
    Join r = {};
    if (j.p.splits > 1) {
        const int64_t want = (j.g.M * ((j.g.N + 7) / 8) + 255) / 256;
        r.splits = j.p.splits;
        r.blocks = (int)(want < 8192 ? want : 8192);
        if (j.g.colsum) { r.sums = j.g.colsum_part; r.parts = j.p.splits; r.n = j.g.M; r.sum_out = j.g.colsum; }
    }
    if (j.sums.sum_out) { r.sums = j.sums.sums; r.parts = j.sums.parts; r.n = j.sums.n; r.sum_out = j.sums.sum_out; }
    r.sum_blocks = r.sum_out ? (int)((r.n + 63) / 64) : 0;
    return r;
}

// one product, or a layer's dx and dw
template <class T>
static int launch_jobs(const Job* jobs, int count, hipStream_t stream)
{
    const Job& a = jobs[0];
    const Job& b = jobs[count - 1];
    const Join ja = join_of(a), jb = count == 2 ? join_of(b) : Join{};
    const int64_t blocks = (int64_t)ja.blocks + ja.sum_blocks + jb.blocks + jb.sum_blocks;
    if (!grid_fits((double)blocks, 256)) return SMLVM_ERR_UNSUPPORTED;
    if (count == 2 && a.p.bm == 64 && b.p.bm == 64) {
        const int64_t blocks_a = (int64_t)a.g.tiles_m * a.g.tiles_n * a.p.splits, blocks_b = (int64_t)b.g.tiles_m * b.g.tiles_n * b.p.splits;
        if (!grid_fits((double)(blocks_a + blocks_b), 256)) return SMLVM_ERR_UNSUPPORTED;
        const dim3 grid((unsigned)(blocks_a + blocks_b));
        if (sizeof(T) == 2 && a.direct && b.direct) {
            if constexpr (sizeof(T) == 2)
                hipLaunchKernelGGL((pair_kernel<T, true>), grid, dim3(256), 0, stream, a.g, b.g, (int)blocks_a);
        } else {
            hipLaunchKernelGGL((pair_kernel<T, false>), grid, dim3(256), 0, stream, a.g, b.g, (int)blocks_a);
        }
    } else {
        for (int i = 0; i < count; ++i) {
            const Job& j = jobs[i];
            if (j.layout == 0) launch_gemm<T, false, false>(j.p, j.direct, j.g, stream);
            else if (j.layout == 1) launch_gemm<T, false, true>(j.p, j.direct, j.g, stream);
            else launch_gemm<T, true, true>(j.p, j.direct, j.g, stream);
        }
    }
    if (blocks) hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, stream, a.g, ja, b.g, jb);
    return check_launch();
}

static int launch_kind(int kind, const Job* jobs, int count, hipStream_t stream)
{
    if (kind == SMLVM_F32) return launch_jobs<float>(jobs, count, stream);
    if (kind == SMLVM_F16) return launch_jobs<f16_t>(jobs, count, stream);
    return launch_jobs<bf16_t>(jobs, count, stream);
}

static size_t workspace_of(int kind, int64_t M, int64_t N, int64_t K, bool colsum)
{
    size_t most = 0;
    for (int direct = 0; direct < 2; ++direct) {     // (which one it is depends on the pointers)
        const Plan p = plan(kind, M, N, K, direct != 0);
        const size_t need = p.splits > 1 ? (size_t)p.splits * M * (N + (colsum ? 1 : 0)) : 0;
        if (need > most) most = need;
    }
    return most * sizeof(float);
}

// dh, in front of the products' partial sums
static size_t act_bytes(int kind, int64_t M, int64_t N) { return ((size_t)M * N * kind_bytes(kind) + 15) & ~(size_t)15; }

// How act_bwd_kernel covers [M, N]: columns by `across` workgroups, rows in `parts`, some 2048 workgroups in all
// with 4 rows at least for a thread.
struct ActPlan {
    int groups;
    int64_t across, parts, rows;
    size_t bytes(int64_t N) const { return ((size_t)parts * N * sizeof(float) + 15) & ~(size_t)15; }
};
static ActPlan act_plan(int64_t M, int64_t N)
{
    ActPlan p = {1, 0, 0, 0};
    if (M <= 0 || N <= 0) return p;
    while (p.groups < 256 && p.groups * 8 < N) p.groups *= 2;
    p.across = (N + p.groups * 8 - 1) / (p.groups * 8);
    const int64_t least = (256 / p.groups) * 4, most = (M + least - 1) / least;
    p.parts = (2048 + p.across - 1) / p.across;
    if (p.parts > most) p.parts = most;
    if (p.parts < 1) p.parts = 1;
    p.rows = (M + p.parts - 1) / p.parts;
    if (p.rows < 1) p.rows = 1;
    p.parts = (M + p.rows - 1) / p.rows;
    return p;
}

// 1: go on, negative: an error
static int check_sizes(int kind, int64_t M, int64_t N, int64_t K)
{
    if (M < 0 || N < 0 || K < 0 || !kind_ok(kind)) return SMLVM_ERR_INVALID;
    if (M > 0x7FFFFFFF || N > 0x7FFFFFFF || K > 0x7FFFFFFF) return SMLVM_ERR_UNSUPPORTED;
    return 1;
}

}  // namespace smlvm

using namespace smlvm;

extern "C" size_t smlvm_linear_fwd_workspace_bytes(int32_t kind, int64_t M, int64_t N, int64_t K)
{
    return check_sizes(kind, M, N, K) == 1 && M > kFewRows ? workspace_of(kind, M, N, K, false) : 0;
}

extern "C" size_t smlvm_linear_bwd_workspace_bytes(int32_t kind, int32_t act, int64_t M, int64_t N, int64_t K)
{
    if (check_sizes(kind, M, N, K) != 1) return 0;
    const size_t dx = workspace_of(kind, M, K, N, false), dw = workspace_of(kind, N, K, M, true);
    return dx + dw + (act ? act_bytes(kind, M, N) + act_plan(M, N).bytes(N) : 0);
}

extern "C" int smlvm_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                const void* residual, int64_t ldr, void* y, void* pre, int32_t kind, int32_t act,
                                int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream)
{
    const int go = check_sizes(kind, M, N, K);
    if (go < 0) return go;
    if (act < kNone || act > kTanh) return SMLVM_ERR_INVALID;
    if (M == 0 || N == 0) return SMLVM_OK;
    if (!y || (K && (!x || !w)) || (K && (ldx < K || ldw < K)) || (residual && ldr < N)) return SMLVM_ERR_INVALID;
    GemmArgs g = {};
    g.a = x; g.b = w; g.lda = ldx; g.ldb = ldw; g.M = M; g.N = N; g.K = K;
    g.out = y; g.bias = bias; g.res = residual; g.ldr = ldr; g.pre = pre; g.act = act;
    if (M <= kFewRows) {
        if (!grid_fits((double)((N + 7) / 8), 256)) return SMLVM_ERR_UNSUPPORTED;
        if (kind == SMLVM_F32) launch_few_rows<float>(g, (hipStream_t)stream);
        else if (kind == SMLVM_F16) launch_few_rows<f16_t>(g, (hipStream_t)stream);
        else launch_few_rows<bf16_t>(g, (hipStream_t)stream);
        return check_launch();
    }
    Job job = {};
    job.g = g;
    char* ws = static_cast<char*>(workspace);
    const int rc = plan_job(job, kind, 0, nullptr, ws, workspace_bytes);
    return rc == SMLVM_OK ? launch_kind(kind, &job, 1, (hipStream_t)stream) : rc;
}

extern "C" int smlvm_linear_bwd(const void* dy, int64_t ldy, const void* h, int32_t h_is_y, const void* x, int64_t ldx,
                                const void* w, int64_t ldw, void* dx, void* dw, void* db, int32_t kind, int32_t act,
                                int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream_)
{
    const int go = check_sizes(kind, M, N, K);
    if (go < 0) return go;
    if (act < kNone || act > kTanh || (h_is_y && act != kRelu) || (db && !dw && K)) return SMLVM_ERR_INVALID;
    const bool some = M && N;                                            // dy is not empty
    if ((some && (!dy || ldy < N || (act && (!h || ldy != N)))) || (dx && N && K && (!w || ldw < K)) ||
        (dw && M && K && (!x || ldx < K))) return SMLVM_ERR_INVALID;
    const hipStream_t stream = (hipStream_t)stream_;
    char* ws = static_cast<char*>(workspace);
    Join sums = {};
    if (act && some) {
        const ActPlan p = act_plan(M, N);
        const size_t held = act_bytes(kind, M, N), bytes = held + (db ? p.bytes(N) : 0);
        if (!ws || workspace_bytes < bytes) return SMLVM_ERR_WORKSPACE;
        float* const part = db ? reinterpret_cast<float*>(ws + held) : nullptr;
        const dim3 grid((unsigned)p.across, (unsigned)p.parts);
#define ACT_BWD(T, H) hipLaunchKernelGGL((act_bwd_kernel<T, H>), grid, dim3(256), 0, stream, static_cast<const T*>(dy), \
                                         static_cast<const H*>(h), reinterpret_cast<T*>(ws), M, N, act, p.groups, p.rows, part)
        if (kind == SMLVM_F32) ACT_BWD(float, float);
        else if (kind == SMLVM_F16 && act == kRelu) ACT_BWD(f16_t, f16_t);             // (y or pre)
        else if (kind == SMLVM_F16) ACT_BWD(f16_t, float);
        else if (h_is_y) ACT_BWD(bf16_t, bf16_t);
        else ACT_BWD(bf16_t, f16_t);
#undef ACT_BWD
        const int rc = check_launch();
        if (rc != SMLVM_OK) return rc;
        if (db) { sums.sums = part; sums.parts = (int)p.parts; sums.n = N; sums.sum_out = db; }
        dy = ws;
        ws += bytes;
        workspace_bytes -= bytes;
    }
    Job jobs[2] = {};
    int count = 0, rc = SMLVM_OK;
    if (dx && M && K) {
        Job& j = jobs[count++];
        j.g.a = dy; j.g.b = w; j.g.lda = ldy; j.g.ldb = ldw; j.g.M = M; j.g.N = K; j.g.K = N; j.g.out = dx;
        rc = plan_job(j, kind, 1, nullptr, ws, workspace_bytes);
    }
    if (rc == SMLVM_OK && N && (K ? dw != nullptr : db != nullptr)) {
        Job& j = jobs[count++];
        j.sums = sums;
        j.g.a = dy; j.g.b = x; j.g.lda = ldy; j.g.ldb = ldx; j.g.M = N; j.g.N = K; j.g.K = M; j.g.out = dw;
        rc = plan_job(j, kind, 2, sums.sum_out ? nullptr : db, ws, workspace_bytes);
    }
    if (rc != SMLVM_OK || count == 0) return rc;
    return launch_kind(kind, jobs, count, stream);
}
