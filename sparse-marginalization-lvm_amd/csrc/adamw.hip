// AdamW over many tensors at once, states in 32 or in 8 bits (formulas: include/sparsemarg.h).
//
// HBM bound: 28 B per element with fp32 weights, gradients and states (read p, g, m, v; write p, m,
// v), 10 B with bf16 weights and gradients and 8-bit states.  Measured: 403M fp32 weights 2.06 ms (5.5 TB/s), 116M
// bf16 weights with 8-bit states 252 us (4.6 TB/s, arithmetic taking about as long).  Small models are launch bound instead,
// so one launch carries up to kTensors tensors: their table travels in the kernel arguments (no
// device table to upload, nothing kept between calls, and a captured launch holds its own copy).
// A workgroup owns kPass * passes consecutive elements of one tensor; a lane owns 8 of them at a time, so
// that 32 lanes hold one 256-element block of an 8-bit state and its maximum is a reduction inside
// half a wave.
#include "elements.hpp"

#include <math.h>

namespace smlvm {

constexpr int kTensors = 40;          // table entries a launch carries (72 B each: 2.9 KB of 4 KB)
constexpr int kThreads = 256;
constexpr int kLane = 8;              // consecutive elements per lane and pass
constexpr int kPass = kThreads * kLane;
constexpr int64_t kMostBlocks = 0xFFFFFF;   // a launch's threads stay below 2^32

struct AdamwTable {
    smlvm_adamw_tensor t[kTensors];
    uint32_t first[kTensors + 1];     // first workgroup of every tensor
    int32_t count;
    int32_t passes;                   // passes of kPass elements per workgroup
};

struct AdamwHyper {
    double beta1, beta2, log2_beta1, log2_beta2;
    const float* lr_dev;
    float eps, lr, weight_decay;
    uint32_t seed;
    uint32_t* ticket;
};

// Multiply-xorshift hash of 32 bits; the multipliers are the odd numbers next to 2^32 (sqrt 5 - 1) / 2
// and 2^32 (sqrt 3 - 1).
constexpr uint32_t kC1 = 0x9E3779B9u, kC2 = 0xBB67AE85u;
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= kC1;
    x ^= x >> 15;
    x *= kC2;
    return x ^ (x >> 16);
}

__device__ __forceinline__ bool finite_f32(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7F800000u) != 0x7F800000u; }

// Exponent k of the smallest scale 2^k, k >= -100, with top <= 448 * 2^k = 1.75 * 2^(k + 8).
__device__ __forceinline__ int scale_exponent(float top)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, top);
    const int e = (int)(b >> 23) - 127;                        // top in [2^e, 2^(e+1)) (zero, subnormal: -127)
    const int k = e - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // mantissa over 1.75: one more
    return k < -100 ? -100 : k;
}
__device__ __forceinline__ float pow2f(int k) { return __builtin_bit_cast(float, (uint32_t)(k + 127) << 23); }

// Square roots of 8 values >= 0, correctly rounded (but for what lies within 2^-46 of a midpoint) in 5
// instructions each: the residual of v rsq(v) is exact in an fma, and half of rsq(v) times it is the correction.
// A wave that holds a zero, a subnormal number, an infinity or a NaN takes sqrtf.
__device__ __forceinline__ void sqrt8(float (&v)[8])
{
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) odd |= __builtin_amdgcn_classf(v[j], 0x2F3);
    if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = sqrtf(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float r = __builtin_amdgcn_rsqf(v[j]);
            const float s = v[j] * r;
            v[j] = fmaf(fmaf(-s, s, v[j]), 0.5f * r, s);
        }
    }
}

// e4m3 code of x * 2^-k, rounded up with probability u16 / 2^16 of the distance (FLOOR: positive values
// keep at least the smallest code).  From 2^-6 on a code is the top of the fp32 pattern: 20 mantissa bits lie
// below it, the random ones are added to the upper 16 of those and the sum cut off, carries into the
// exponent included.  Below, codes are 2^-9 apart.
template <bool FLOOR>
__device__ __forceinline__ uint32_t encode_e4m3(float x, float inv_scale, uint32_t u16)
{
    const float y = fabsf(x) * inv_scale;
    const uint32_t raw = ((__builtin_bit_cast(uint32_t, y) + (u16 << 4)) >> 20) - (120u << 3);
    const uint32_t low = (uint32_t)fmaf(y, 512.0f, (float)u16 * 0x1p-16f);
    uint32_t code = y < 0x1p-6f ? low : raw > 0x7Eu ? 0x7Eu : raw;
    if constexpr (FLOOR) code = code == 0 && y > 0.0f ? 1u : code;
    if (!finite_f32(x)) code = 0x7F;
    return code | (FLOOR ? 0u : (__builtin_bit_cast(uint32_t, x) >> 24) & 0x80u);
}

// Largest finite |x| of 8 values in each of 32 lanes: fmaxf passes NaN over, infinities are sorted out where
// there are any.
__device__ __forceinline__ float block_top(const float (&x)[8])
{
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
    top = group_reduce<32>(top, OpMaxF{});
    if (__builtin_amdgcn_ballot_w64(!finite_f32(top)) != 0) {     // (uniform: the whole wave takes it)
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) t = finite_f32(x[j]) ? fmaxf(t, fabsf(x[j])) : t;
        top = group_reduce<32>(t, OpMaxF{});
    }
    return top;
}

__device__ __forceinline__ void decode_e4m3(u32x2 codes, float scale, float (&x)[8])
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], true);
        x[4 * w + 0] = lo.x * scale;
        x[4 * w + 1] = lo.y * scale;
        x[4 * w + 2] = hi.x * scale;
        x[4 * w + 3] = hi.y * scale;
    }
}

template <class T>
__device__ __forceinline__ void load_some(const T* p, int have, float (&x)[8])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < have ? (float)p[j] : 0.0f;
}
template <class T>
__device__ __forceinline__ void store_some(T* p, int have, const float (&x)[8])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < have) p[j] = (T)x[j];
}
__device__ __forceinline__ u32x2 load_codes(const uint8_t* p, int have, bool whole)
{
    if (whole) return *reinterpret_cast<const u32x2*>(p);
    u32x2 r = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < have) r[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
    return r;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int have, bool whole, u32x2 c)
{
    if (whole) { *reinterpret_cast<u32x2*>(p) = c; return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < have) p[j] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
}

template <class PT, class GT, int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const AdamwTable table, const AdamwHyper hp)
{
    int ti = 0;
    for (int lo = 0, hi = table.count; hi - lo > 1;) {          // wave-uniform: the tensor of this workgroup
        const int mid = (lo + hi) >> 1;
        if (blockIdx.x >= table.first[mid]) lo = mid; else hi = mid;
        ti = lo;
    }
    const smlvm_adamw_tensor& t = table.t[ti];
    const int64_t begin = (int64_t)(blockIdx.x - table.first[ti]) * table.passes * kPass;
    PT* const p_ = static_cast<PT*>(t.p);
    const GT* const g_ = static_cast<const GT*>(t.g);
    const int64_t step = *t.step + 1;
    const float lr = hp.lr_dev ? *hp.lr_dev : hp.lr;
    // 16-byte accesses need aligned tensors (views into a flat buffer may start anywhere)
    const bool aligned = (((uintptr_t)t.p | (uintptr_t)t.g | (uintptr_t)t.m | (uintptr_t)t.v) & 15u) == 0;

    const float correct1 = (float)(1.0 - exp2((double)step * hp.log2_beta1));
    const float rsqrt2 = (float)(1.0 / sqrt(1.0 - exp2((double)step * hp.log2_beta2)));
    const float step_size = lr / correct1, keep = 1.0f - lr * hp.weight_decay;
    const uint32_t key0 = mix(mix(hp.seed + kC1 * (uint32_t)step) + (uint32_t)t.index);
    const float b1 = (float)hp.beta1, b2 = (float)hp.beta2;
    const float c1 = (float)(1.0 - hp.beta1), c2 = (float)(1.0 - hp.beta2);

    for (int pass = 0; pass < table.passes; ++pass) {
        const int64_t at = begin + (int64_t)pass * kPass + threadIdx.x * kLane;
        if (begin + (int64_t)pass * kPass >= t.n) break;         // (workgroup-uniform)
        const int64_t left = t.n - at;
        const int have = left <= 0 ? 0 : left < kLane ? (int)left : kLane;
        const bool whole = aligned && have == kLane;
        float p[8], g[8], m[8], v[8];
        if (whole) {
            load_vec(p_ + at, p);
            load_vec(g_ + at, g);
        } else {
            load_some(p_ + at, have, p);
            load_some(g_ + at, have, g);
        }
        if constexpr (BITS == 32) {
            float* const m_ = static_cast<float*>(t.m) + at;
            float* const v_ = static_cast<float*>(t.v) + at;
            if (whole) { load_vec(m_, m); load_vec(v_, v); }
            else { load_some(m_, have, m); load_some(v_, have, v); }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m[j] = fmaf(b1, m[j], c1 * g[j]);
                v[j] = fmaf(b2, v[j], c2 * (g[j] * g[j]));
            }
            if (whole) { store_vec(m_, m); store_vec(v_, v); }
            else { store_some(m_, have, m); store_some(v_, have, v); }
            sqrt8(v);
        } else {
            uint8_t* const m_ = static_cast<uint8_t*>(t.m) + at;
            uint8_t* const r_ = static_cast<uint8_t*>(t.v) + at;
            const int64_t block = at >> 8;                       // 32 lanes share it
            const float ms = have ? t.m_scale[block] : 0.0f, rs = have ? t.r_scale[block] : 0.0f;
            decode_e4m3(load_codes(m_, have, whole), ms, m);
            decode_e4m3(load_codes(r_, have, whole), rs, v);
            // fp64 averages, rounded once: which code and which scale a value gets then does not depend
            // on how its sum was associated
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double gd = (double)g[j], rd = (double)v[j];
                m[j] = (float)fma(hp.beta1, (double)m[j], (1.0 - hp.beta1) * gd);
                v[j] = (float)fma(hp.beta2, rd * rd, (1.0 - hp.beta2) * (gd * gd));
            }
            sqrt8(v);
            const int mk = scale_exponent(block_top(m)), rk = scale_exponent(block_top(v));
            const float minv = pow2f(-mk), rinv = pow2f(-rk);
            u32x2 mc = {0u, 0u}, rc = {0u, 0u};
            const uint32_t key = key0 + (uint32_t)((uint64_t)at >> 32);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t u = mix(((uint32_t)at + j) * kC1 + key);
                mc[j >> 2] |= encode_e4m3<false>(m[j], minv, u & 0xFFFFu) << (8 * (j & 3));
                rc[j >> 2] |= encode_e4m3<true>(v[j], rinv, u >> 16) << (8 * (j & 3));
            }
            store_codes(m_, have, whole, mc);
            store_codes(r_, have, whole, rc);
            if ((threadIdx.x & 31) == 0 && have) {
                t.m_scale[block] = pow2f(mk);
                t.r_scale[block] = pow2f(rk);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)                              // v holds sqrt(v) here
            // (the hardware's reciprocal, 1 ulp, for a division of ten instructions)
            p[j] = fmaf(-step_size, m[j] * __builtin_amdgcn_rcpf(fmaf(v[j], rsqrt2, hp.eps)), p[j] * keep);
        if (whole) store_vec(p_ + at, p); else store_some(p_ + at, have, p);
    }

    // Every workgroup has read its step before it takes a number here (nothing else is ordered by the
    // ticket, so it is relaxed: a release would write the whole L2 back); the last one counts all
    // the launch's tensors up and hands the ticket back at zero.  A captured launch has no ticket: its word would have
    // to outlive every graph that holds it, and two graphs replayed side by side would share it.
    if (hp.ticket == nullptr) return;                            // (a kernel of its own counts up)
    __syncthreads();
    if (threadIdx.x == 0) {
        if (__hip_atomic_fetch_add(hp.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
            for (int i = 0; i < table.count; ++i) *table.t[i].step += 1;
            __hip_atomic_store(hp.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

__global__ __launch_bounds__(64) void count_up_kernel(const AdamwTable table)
{
    if ((int)threadIdx.x < table.count) *table.t[threadIdx.x].step += 1;
}

template <class PT, class GT>
static void launch(int bits, const AdamwTable& table, const AdamwHyper& hp, uint32_t blocks, hipStream_t stream)
{
    if (bits == 32) hipLaunchKernelGGL((adamw_kernel<PT, GT, 32>), dim3(blocks), dim3(kThreads), 0, stream, table, hp);
    else hipLaunchKernelGGL((adamw_kernel<PT, GT, 8>), dim3(blocks), dim3(kThreads), 0, stream, table, hp);
}

template <class PT>
static void launch_g(int g_kind, int bits, const AdamwTable& table, const AdamwHyper& hp, uint32_t blocks, hipStream_t stream)
{
    if (g_kind == SMLVM_F32) launch<PT, float>(bits, table, hp, blocks, stream);
    else if (g_kind == SMLVM_F16) launch<PT, f16_t>(bits, table, hp, blocks, stream);
    else launch<PT, bf16_t>(bits, table, hp, blocks, stream);
}

}  // namespace smlvm

using namespace smlvm;

extern "C" int smlvm_adamw_step(const smlvm_adamw_tensor* tensors, int32_t count, int32_t p_kind, int32_t g_kind,
                                int32_t state_bits, double beta1, double beta2, float eps, float lr,
                                const float* lr_dev, float weight_decay, uint32_t seed, uint32_t* ticket,
                                void* stream)
{
    if (count < 0 || !kind_ok(p_kind) || !kind_ok(g_kind) || (state_bits != 32 && state_bits != 8)) return SMLVM_ERR_INVALID;
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return SMLVM_ERR_INVALID;
    if (count == 0) return SMLVM_OK;
    uint64_t capture = 0;
    const int asked = smlvm_stream_capture_id(stream, &capture);
    if (asked != SMLVM_OK) return asked;
    if (!tensors || (!ticket && !capture)) return SMLVM_ERR_INVALID;
    int64_t most = 0;
    for (int i = 0; i < count; ++i) {
        const smlvm_adamw_tensor& t = tensors[i];
        if (t.n < 0) return SMLVM_ERR_INVALID;
        if (t.n && (!t.p || !t.g || !t.m || !t.v || !t.step)) return SMLVM_ERR_INVALID;
        if (t.n && state_bits == 8 && (!t.m_scale || !t.r_scale)) return SMLVM_ERR_INVALID;
        if (t.n > kMostBlocks * kPass) return SMLVM_ERR_UNSUPPORTED;
        most += t.n;
    }
    AdamwHyper hp;
    hp.beta1 = beta1; hp.beta2 = beta2;
    hp.log2_beta1 = log2(beta1); hp.log2_beta2 = log2(beta2);          // (-inf for 0: beta^t = 0)
    hp.lr_dev = lr_dev; hp.eps = eps; hp.lr = lr; hp.weight_decay = weight_decay;
    hp.seed = seed; hp.ticket = ticket;
    AdamwTable table;
    // A workgroup's fixed cost (finding its tensor, two fp64 powers) is paid once per `passes` passes; but one pass's
    // stores and the next one's loads do not overlap, other workgroups' do.  fp32 states: 1 pass 2.06 ms, 2 passes 2.11,
    // up to 48 passes 2.30 (403M weights).  8-bit states, which are bound by arithmetic: 1 pass 291 us, 2 271, 8 260,
    // 13 265 (117M weights).
    const int64_t most_passes = state_bits == 32 ? 1 : 8, passes = most / ((int64_t)kPass * 4096);
    table.passes = (int32_t)(passes < 1 ? 1 : passes > most_passes ? most_passes : passes);
    const int64_t chunk = (int64_t)kPass * table.passes;
    for (int i = 0; i < count;) {
        table.count = 0;
        uint64_t blocks = 0;
        for (; i < count && table.count < kTensors; ++i) {
            if (tensors[i].n == 0) continue;
            const uint64_t need = (uint64_t)((tensors[i].n + chunk - 1) / chunk);
            if (blocks + need > kMostBlocks && table.count) break;
            table.t[table.count] = tensors[i];
            table.first[table.count++] = (uint32_t)blocks;
            blocks += need;
        }
        if (!table.count) break;
        table.first[table.count] = (uint32_t)blocks;
        // One word takes some 12 ns per workgroup: from 4096 on a second launch is cheaper.
        hp.ticket = blocks <= 4096 && !capture ? ticket : nullptr;
        if (p_kind == SMLVM_F32) launch_g<float>(g_kind, state_bits, table, hp, (uint32_t)blocks, (hipStream_t)stream);
        else if (p_kind == SMLVM_F16) launch_g<f16_t>(g_kind, state_bits, table, hp, (uint32_t)blocks, (hipStream_t)stream);
        else launch_g<bf16_t>(g_kind, state_bits, table, hp, (uint32_t)blocks, (hipStream_t)stream);
        if (!hp.ticket) hipLaunchKernelGGL(count_up_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, table);
        const int rc = check_launch();
        if (rc != SMLVM_OK) return rc;
    }
    return SMLVM_OK;
}
