// Log-probabilities of chosen tokens, their backward, and the clipped policy loss whose gradient with
// respect to the logits is written in the pass that reads them (formulas: include/sparsemarg.h).
//
// HBM bound: the floor is one read of the logits and, for training, one write of as many bytes.
// A row is held by one lane group (8 lanes ... 1024 threads) in registers, 16 bytes per lane and
// vector, so that the softmax statistics and the gradient need a single read; rows too long for 32
// vectors per thread (512 of them) are read twice by the same workgroup, the second time out of the caches.
// Measured: log-probabilities of [8192 x 65536] bf16 181 us (5.9 TB/s); the loss of [8192 x 128000] bf16 with its
// gradient, about half of the rows masked, 840 us.
//
// Softmax statistics in one pass: y_j = (z_j - m) log2 e with m the running maximum; s = sum 2^y_j and
// t = sum 2^y_j y_j are rescaled when m moves, by d = (m_old - m_new) log2 e <= 0:
//     t <- 2^d (t + d s),   s <- 2^d s.
// Then p_j = 2^y_j / s, log p_j = (y_j - log2 s) ln 2, entropy = ln 2 (log2 s - t / s).  (z - m first: one
// fma(z, log2 e, -m log2 e) would overflow for rows at the type's lowest value, which are uniform.)
// The gradient c (1[j = a] - p_j) - h p_j (log p_j + H) = c 1[j = a] - 2^y_j (A + B y_j) with
// A = (c + h (H - ln s)) / s and B = h ln 2 / s.
#include "elements.hpp"

#include <math.h>

namespace smlvm {

constexpr float kL = 1.44269504088896340736f;        // log2 e
constexpr double kLn2d = 0.693147180559945309417;
constexpr float kLowest = -3.40282346638528859812e38f;   // "no maximum yet": finite, so that s = 0 stays 0

typedef u32x4 __attribute__((aligned(2))) u32x4_any;  // rows may start at any element

__device__ __forceinline__ float ex2f(float v) { return __builtin_amdgcn_exp2f(v); }

template <class T> __device__ __forceinline__ constexpr uint32_t neg_inf_word();
template <> __device__ __forceinline__ constexpr uint32_t neg_inf_word<float>() { return 0xFF800000u; }
template <> __device__ __forceinline__ constexpr uint32_t neg_inf_word<f16_t>() { return 0xFC00FC00u; }
template <> __device__ __forceinline__ constexpr uint32_t neg_inf_word<bf16_t>() { return 0xFF80FF80u; }

template <class T> constexpr int kPer = 16 / (int)sizeof(T);     // elements per vector

// vector v of a row of V elements; what lies beyond the row is -inf (probability 0)
template <class T>
__device__ __forceinline__ u32x4 load_row_vec(const T* __restrict__ z, int v, int V)
{
    constexpr int P = kPer<T>;
    const int64_t at = (int64_t)v * P;
    constexpr uint32_t w = neg_inf_word<T>();
    u32x4 raw = {w, w, w, w};
    if (at + P <= V) {
        raw = *reinterpret_cast<const u32x4_any*>(z + at);
    } else if (at < V) {
        T t[P];
        __builtin_memcpy(t, &raw, 16);
#pragma unroll
        for (int j = 0; j < P; ++j) if (at + j < V) t[j] = z[at + j];
        __builtin_memcpy(&raw, t, 16);
    }
    return raw;
}

template <class T>
__device__ __forceinline__ void unpack(u32x4 raw, float (&x)[kPer<T>])
{
    T t[kPer<T>];
    __builtin_memcpy(t, &raw, 16);
#pragma unroll
    for (int j = 0; j < kPer<T>; ++j) x[j] = (float)t[j];
}

template <class T>
__device__ __forceinline__ void store_row_vec(T* __restrict__ d, int v, int V, const float (&x)[kPer<T>])
{
    constexpr int P = kPer<T>;
    const int64_t at = (int64_t)v * P;
    T t[P];
#pragma unroll
    for (int j = 0; j < P; ++j) t[j] = (T)x[j];
    if (at + P <= V) {
        u32x4 raw;
        __builtin_memcpy(&raw, t, 16);
        *reinterpret_cast<u32x4_any*>(d + at) = raw;
    } else if (at < V) {
#pragma unroll
        for (int j = 0; j < P; ++j) if (at + j < V) d[at + j] = t[j];
    }
}

struct Stats { float m, s, t; };

__device__ __forceinline__ void rescale(Stats& a, float m)
{
    const float d = fmaxf(a.m - m, -1e30f) * kL;      // (finite, for d * 0)
    const float f = ex2f(d);
    a.t = f * fmaf(d, a.s, a.t);
    a.s *= f;
    a.m = m;
}

// N elements more
template <int N>
__device__ __forceinline__ void absorb(Stats& a, const float (&z)[N])
{
    float top = z[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, z[j]);
    const float m = fmaxf(a.m, top);
    if (m != a.m) rescale(a, m);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float y = (z[j] - m) * kL;
        const float e = ex2f(y);
        a.s += e;
        a.t = fmaf(e, fmaxf(y, -1000.0f), a.t);      // (0 * -inf would be NaN; a NaN reaches s through e)
    }
}

struct RowsIn {
    const void* z;
    int64_t stride_b, stride_t;
    const int64_t* actions;
    const uint8_t* mask;
    uint32_t rows, T;
    int32_t V;
};
struct RowsOut {
    float *logp, *entropy, *stats;
    void* dz;
};
struct Policy {
    const float *old_logp, *adv, *ref;
    double low, high, kl_coeff, ent_coeff, norm;
    const double* norm_dev;       // instead of norm
    float *kl, *c, *h;
    uint8_t* clipped;
    double* row_loss;
};

template <class T>
__device__ __forceinline__ const T* row_of(const RowsIn& in, uint32_t row)
{
    const uint32_t b = row / in.T, t = row - b * in.T;
    return static_cast<const T*>(in.z) + (int64_t)b * in.stride_b + (int64_t)t * in.stride_t;
}

// What one row's gradient needs: A, B, c (above).
struct Slope { float A, B, c; };

// The scalars of one row, computed by one lane.  fp64: three log / exp per row cost nothing next to
// the row, and e^d - d - 1 cancels for small d.
template <bool POLICY>
__device__ Slope finish_row(const RowsIn& in, const RowsOut& out, const Policy& pol, uint32_t row, bool live,
                            bool on, int64_t action, float za, const Stats& st)
{
    Slope sl = {0.0f, 0.0f, 0.0f};
    if (!live) return sl;
    double logp = 0.0, ent = 0.0, loss = 0.0, kl = 0.0, c = 0.0, h = 0.0;
    bool clip = false;
    if (on) {
        const double ls = log2((double)st.s);
        ent = kLn2d * (ls - (double)st.t / (double)st.s);
        logp = (double)za - (double)st.m - kLn2d * ls;
        if (action < 0 || action >= in.V) logp = __builtin_nan("");
        if constexpr (POLICY) {
            const double norm = pol.norm_dev ? *pol.norm_dev : pol.norm;
            const double adv = pol.adv[row];
            const double ratio = exp(logp - (double)pol.old_logp[row]);
            clip = (adv > 0.0 && ratio > 1.0 + pol.high) || (adv < 0.0 && ratio < 1.0 - pol.low);
            const double used = clip ? (adv > 0.0 ? 1.0 + pol.high : 1.0 - pol.low) : ratio;
            loss = -used * adv - pol.ent_coeff * ent;
            c = clip ? 0.0 : -adv * ratio;
            if (pol.ref) {
                const double d = (double)pol.ref[row] - logp;
                const double grow = expm1(d);
                kl = grow - d;
                loss += pol.kl_coeff * kl;
                c -= pol.kl_coeff * grow;
            }
            c *= norm;
            h = -pol.ent_coeff * norm;
        }
        const double inv = 1.0 / (double)st.s;
        sl.c = (float)c;
        sl.A = (float)((c + h * (ent - kLn2d * ls)) * inv);
        sl.B = (float)(h * kLn2d * inv);
    }
    if (out.logp) out.logp[row] = (float)logp;
    if (out.entropy) out.entropy[row] = (float)ent;
    if (out.stats) {
        out.stats[3 * (int64_t)row] = on ? st.m : 0.0f;
        out.stats[3 * (int64_t)row + 1] = on ? st.s : 1.0f;
        out.stats[3 * (int64_t)row + 2] = (float)ent;
    }
    if constexpr (POLICY) {
        pol.row_loss[row] = loss;
        pol.c[row] = (float)c;
        pol.h[row] = (float)h;
        if (pol.kl) pol.kl[row] = (float)kl;
        if (pol.clipped) pol.clipped[row] = clip ? 1 : 0;
    }
    return sl;
}

template <class T>
__device__ __forceinline__ void gradient_vec(u32x4 raw, T* __restrict__ dz, int v, int V, float m, const Slope& sl,
                                             int64_t action)
{
    constexpr int P = kPer<T>;
    float x[P];
    unpack<T>(raw, x);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const float y = fmaxf((x[j] - m) * kL, -150.0f);     // (2^-150 is 0; -inf * B would be NaN)
        x[j] = -ex2f(y) * fmaf(sl.B, y, sl.A);
    }
    const int64_t at = action - (int64_t)v * P;
    if (at >= 0 && at < P) {
#pragma unroll
        for (int j = 0; j < P; ++j) if (at == j) x[j] += sl.c;
    }
    store_row_vec<T>(dz, v, V, x);
}

// G lanes per row, R vectors per lane in registers; R = 0: the row is streamed twice.
template <class T, int G, int R, bool POLICY, bool GRAD>
__global__ __launch_bounds__(G < 256 ? 256 : G) void rows_kernel(const RowsIn in, const RowsOut out, const Policy pol)
{
    constexpr int BLOCK = G < 256 ? 256 : G;
    constexpr int P = kPer<T>;
    constexpr int U = R == 0 ? 4 : (R < 4 ? R : 4);     // vectors absorbed under one maximum
    uint32_t row = (blockIdx.y * gridDim.x + blockIdx.x) * (BLOCK / G) + threadIdx.x / G;
    const bool live = row < in.rows;
    if (!live) row = in.rows - 1;                        // whole lane groups stay busy
    const int lane = threadIdx.x & (G - 1);
    const T* const z = row_of<T>(in, row);
    const bool on = in.mask ? in.mask[row] != 0 : true;
    const int64_t action = in.actions[row];
    float za = 0.0f;
    if (on && lane == 0 && action >= 0 && action < in.V) za = (float)z[action];
    const int V = on ? in.V : 0;                         // a masked row is not read

    u32x4 keep[R > 0 ? R : 1];
    Stats st = {kLowest, 0.0f, 0.0f};
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) keep[i] = load_row_vec<T>(z, lane + i * G, V);
#pragma unroll
        for (int i = 0; i < R; i += U) {
            float x[U * P];
#pragma unroll
            for (int k = 0; k < U; ++k) unpack<T>(keep[i + k], *reinterpret_cast<float(*)[P]>(&x[k * P]));
            absorb(st, x);
        }
    } else {
        for (int64_t v = lane; v * P < V; v += (int64_t)U * G) {
            float x[U * P];
#pragma unroll
            for (int k = 0; k < U; ++k)
                unpack<T>(load_row_vec<T>(z, (int)v + k * G, V), *reinterpret_cast<float(*)[P]>(&x[k * P]));
            absorb(st, x);
        }
    }
    rescale(st, group_reduce<G < 64 ? G : 64>(st.m, OpMaxF{}));
    st.s = group_reduce<G < 64 ? G : 64>(st.s, OpSum{});
    st.t = group_reduce<G < 64 ? G : 64>(st.t, OpSum{});

    __shared__ Stats wave_stats[G > 64 ? G / 64 : 1];
    __shared__ Slope shared_slope;
    Slope sl;
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) wave_stats[threadIdx.x >> 6] = st;
        __syncthreads();
        float m = wave_stats[0].m;
#pragma unroll
        for (int w = 1; w < G / 64; ++w) m = fmaxf(m, wave_stats[w].m);
        st = {m, 0.0f, 0.0f};
        for (int w = 0; w < G / 64; ++w) {
            Stats other = wave_stats[w];
            rescale(other, m);
            st.s += other.s;
            st.t += other.t;
        }
        if (threadIdx.x == 0) shared_slope = finish_row<POLICY>(in, out, pol, row, live, on, action, za, st);
        if constexpr (GRAD) {
            __syncthreads();
            sl = shared_slope;
        }
    } else {
        if (lane == 0) sl = finish_row<POLICY>(in, out, pol, row, live, on, action, za, st);
        if constexpr (GRAD) {
            sl.A = __shfl(sl.A, 0, G);
            sl.B = __shfl(sl.B, 0, G);
            sl.c = __shfl(sl.c, 0, G);
        }
    }
    if constexpr (GRAD) {
        if (!live) return;
        T* const dz = static_cast<T*>(out.dz) + (int64_t)row * in.V;
        if (!on) {
            float zero[P] = {};
            for (int64_t v = lane; v * P < in.V; v += G) store_row_vec<T>(dz, (int)v, in.V, zero);
            return;
        }
        if constexpr (R > 0) {
            // (opaque: without it the compiler keeps the first pass's unpacked fp32 values instead of
            // the packed ones, twice the registers, and spills)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                asm volatile("" : "+v"(keep[i]));
                gradient_vec<T>(keep[i], dz, lane + i * G, V, st.m, sl, action);
                if constexpr (R >= 8) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            for (int64_t v = lane; v * P < V; v += G)
                gradient_vec<T>(load_row_vec<T>(z, (int)v, V), dz, (int)v, V, st.m, sl, action);
        }
    }
}

// The backward from saved statistics.  Workgroups go over (row or group of rows, part of a long row) units; a
// bounded number of them, so that the call that has nothing to write (keep_if_one) is over at once (65536
// workgroups took 16 us to find out).
template <class T, int G>
__global__ __launch_bounds__(256) void rows_bwd_kernel(const RowsIn in, const float* __restrict__ stats,
                                                       const float* __restrict__ c_, const float* __restrict__ h_,
                                                       const float* __restrict__ g_, int keep_if_one,
                                                       T* __restrict__ out, uint32_t units, uint32_t parts)
{
    constexpr int P = kPer<T>;
    const float g = g_ ? *g_ : 1.0f;
    if (keep_if_one && g == 1.0f) return;
    const int lane = threadIdx.x & (G - 1);
    for (uint32_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const uint32_t row = (unit / parts) * (256 / G) + threadIdx.x / G, part = unit % parts;
        if (row >= in.rows) continue;
        T* const dz = out + (int64_t)row * in.V;
        const int64_t first = (int64_t)part * G + lane, step = (int64_t)parts * G;
        if (in.mask && in.mask[row] == 0) {
            float zero[P] = {};
            for (int64_t v = first; v * P < in.V; v += step) store_row_vec<T>(dz, (int)v, in.V, zero);
            continue;
        }
        const T* const z = row_of<T>(in, row);
        const float m = stats[3 * (int64_t)row], s = stats[3 * (int64_t)row + 1], ent = stats[3 * (int64_t)row + 2];
        const float inv = 1.0f / s;
        const float c = g * c_[row], h = h_ ? g * h_[row] : 0.0f;
        const float ln2 = (float)kLn2d;
        const Slope sl = {h_ ? (c + h * (ent - ln2 * log2f(s))) * inv : c * inv, h * ln2 * inv, c};
        const int64_t action = in.actions[row];
        for (int64_t v = first; v * P < in.V; v += step)
            gradient_vec<T>(load_row_vec<T>(z, (int)v, in.V), dz, (int)v, in.V, m, sl, action);
    }
}

// norm = 1 / max(1, number of rows that count)
__global__ __launch_bounds__(1024) void count_kernel(const uint8_t* __restrict__ mask, uint32_t rows, double* norm)
{
    int n = 0;
    for (uint32_t i = threadIdx.x; i < rows; i += 1024) n += mask[i] != 0;
    n = group_reduce<64>(n, OpSum{});
    __shared__ int part[16];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < 16; ++w) all += part[w];
        *norm = 1.0 / (all > 0 ? all : 1);
    }
}

__global__ __launch_bounds__(1024) void sum_kernel(const double* __restrict__ row_loss, uint32_t rows, double norm,
                                                   const double* __restrict__ norm_dev, float* __restrict__ loss)
{
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
    s = group_reduce<64>(s, OpSum{});
    __shared__ double part[16];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < 16; ++w) all += part[w];
        *loss = (float)(all * (norm_dev ? *norm_dev : norm));
    }
}

template <class T, bool POLICY, bool GRAD>
static void launch_rows(const RowsIn& in, const RowsOut& out, const Policy& pol, hipStream_t stream)
{
    const int64_t nv = ((int64_t)in.V + kPer<T> - 1) / kPer<T>;
    // (in two axes: a launch's threads along one of them stay below 2^32)
    auto grid = [&](uint32_t per) {
        const uint32_t blocks = (in.rows + per - 1) / per, x = blocks < (1u << 21) ? blocks : 1u << 21;
        return dim3(x, (blocks + x - 1) / x);
    };
#define ROWS(G, R)                                                                                             \
    hipLaunchKernelGGL((rows_kernel<T, G, R, POLICY, GRAD>), grid(G < 256 ? 256 / G : 1), dim3(G < 256 ? 256 : G), \
                       0, stream, in, out, pol)
    if (nv <= 8) ROWS(8, 1);
    else if (nv <= 64) ROWS(64, 1);
    else if (nv <= 128) ROWS(64, 2);
    else if (nv <= 256) ROWS(64, 4);
    else if (nv <= 512) ROWS(256, 2);
    else if (nv <= 1024) ROWS(256, 4);
    else if (nv <= 2048) ROWS(256, 8);
    else if (nv <= 4096) ROWS(512, 8);
    else if (nv <= 8192) ROWS(512, 16);
    else if (nv <= 16384) ROWS(512, 32);
    else ROWS(1024, 0);
#undef ROWS
}

template <class T>
static void launch_bwd(const RowsIn& in, const float* stats, const float* c, const float* h, const float* g,
                       int keep, void* dz, hipStream_t stream)
{
    const int64_t nv = ((int64_t)in.V + kPer<T> - 1) / kPer<T>;
    const int group = nv <= 8 ? 8 : nv <= 128 ? 64 : 256;
    const int64_t row_units = ((int64_t)in.rows * group + 255) / 256;
    int64_t parts = 1;                                   // few long rows: parts of at least 4 vectors per thread
    if (group == 256 && row_units < 2048) {
        parts = (2048 + row_units - 1) / row_units;
        const int64_t most = (nv + 1023) / 1024;
        if (parts > most) parts = most;
    }
    const int64_t units = row_units * parts;
    const dim3 grid((unsigned)(units < 4096 ? units : 4096));
#define ROWS_BWD(G)                                                                                              \
    hipLaunchKernelGGL((rows_bwd_kernel<T, G>), grid, dim3(256), 0, stream, in, stats, c, h, g, keep,            \
                       static_cast<T*>(dz), (uint32_t)units, (uint32_t)parts)
    if (group == 8) ROWS_BWD(8);
    else if (group == 64) ROWS_BWD(64);
    else ROWS_BWD(256);
#undef ROWS_BWD
}

// 0: nothing to do, 1: go on, negative: an error
static int check_rows(const void* z, int kind, const int64_t* actions, int64_t B, int64_t T, int64_t V)
{
    if (B < 0 || T < 0 || V < 1 || !kind_ok(kind)) return SMLVM_ERR_INVALID;
    if (B == 0 || T == 0) return 0;
    if (!z || !actions) return SMLVM_ERR_INVALID;
    if (B > 0x7FFFFFFF || T > 0x7FFFFFFF || B * T > 0x7FFFFFFF || V > 0x7FFF0000) return SMLVM_ERR_UNSUPPORTED;
    return 1;
}

}  // namespace smlvm

using namespace smlvm;

extern "C" int smlvm_token_logprobs_fwd(const void* logits, int32_t kind, int64_t stride_b, int64_t stride_t,
                                        const int64_t* actions, const uint8_t* mask, float* logp, float* entropy,
                                        float* stats, int64_t B, int64_t T, int64_t V, void* stream)
{
    const int go = check_rows(logits, kind, actions, B, T, V);
    if (go <= 0) return go;
    const RowsIn in = {logits, stride_b, stride_t, actions, mask, (uint32_t)(B * T), (uint32_t)T, (int32_t)V};
    const RowsOut out = {logp, entropy, stats, nullptr};
    const Policy none = {};
    if (kind == SMLVM_F32) launch_rows<float, false, false>(in, out, none, (hipStream_t)stream);
    else if (kind == SMLVM_F16) launch_rows<f16_t, false, false>(in, out, none, (hipStream_t)stream);
    else launch_rows<bf16_t, false, false>(in, out, none, (hipStream_t)stream);
    return check_launch();
}

extern "C" int smlvm_token_logprobs_bwd(const void* logits, int32_t kind, int64_t stride_b, int64_t stride_t,
                                        const int64_t* actions, const uint8_t* mask, const float* stats,
                                        const float* c, const float* h, const float* g, int32_t keep_if_one, void* dlogits, int64_t B, int64_t T, int64_t V,
                                        void* stream)
{
    const int go = check_rows(logits, kind, actions, B, T, V);
    if (go <= 0) return go;
    if (!stats || !c || !dlogits || (keep_if_one && !g)) return SMLVM_ERR_INVALID;
    const RowsIn in = {logits, stride_b, stride_t, actions, mask, (uint32_t)(B * T), (uint32_t)T, (int32_t)V};
    if (kind == SMLVM_F32) launch_bwd<float>(in, stats, c, h, g, keep_if_one, dlogits, (hipStream_t)stream);
    else if (kind == SMLVM_F16) launch_bwd<f16_t>(in, stats, c, h, g, keep_if_one, dlogits, (hipStream_t)stream);
    else launch_bwd<bf16_t>(in, stats, c, h, g, keep_if_one, dlogits, (hipStream_t)stream);
    return check_launch();
}

extern "C" size_t smlvm_policy_loss_workspace_bytes(int64_t rows) { return 8 * (size_t)((rows > 0 ? rows : 0) + 1); }

extern "C" int smlvm_policy_loss(const void* logits, int32_t kind, int64_t stride_b, int64_t stride_t,
                                 const int64_t* actions, const uint8_t* mask, const float* old_logp,
                                 const float* advantages, const float* ref_logp, float clip_low, float clip_high,
                                 float kl_coeff, float entropy_coeff, int32_t mean, float* loss, float* logp,
                                 float* entropy, float* kl, uint8_t* clipped, float* stats, float* c, float* h,
                                 void* dlogits, int64_t B, int64_t T, int64_t V, void* workspace,
                                 size_t workspace_bytes, void* stream_)
{
    const int go = check_rows(logits, kind, actions, B, T, V);
    if (go < 0) return go;
    if (!loss || !(clip_low >= 0.0f) || !(clip_high >= 0.0f)) return SMLVM_ERR_INVALID;
    if (go && (!old_logp || !advantages || !stats || !c || !h)) return SMLVM_ERR_INVALID;
    const int64_t rows = go ? B * T : 0;
    if (!workspace || workspace_bytes < smlvm_policy_loss_workspace_bytes(rows)) return SMLVM_ERR_WORKSPACE;
    const hipStream_t stream = (hipStream_t)stream_;
    double* const ws = static_cast<double*>(workspace);          // [0] norm, [1 ...] the rows' losses
    Policy pol = {};
    pol.old_logp = old_logp; pol.adv = advantages; pol.ref = ref_logp;
    pol.low = clip_low; pol.high = clip_high; pol.kl_coeff = kl_coeff; pol.ent_coeff = entropy_coeff;
    pol.norm = mean ? 1.0 / (rows > 0 ? (double)rows : 1.0) : 1.0;
    pol.norm_dev = mean && mask && rows ? ws : nullptr;
    pol.kl = kl; pol.c = c; pol.h = h; pol.clipped = clipped; pol.row_loss = ws + 1;
    if (pol.norm_dev) hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, stream, mask, (uint32_t)rows, ws);
    if (rows) {
        const RowsIn in = {logits, stride_b, stride_t, actions, mask, (uint32_t)rows, (uint32_t)T, (int32_t)V};
        const RowsOut out = {logp, entropy, stats, dlogits};
#define POLICY_ROWS(TYPE)                                                       \
        do {                                                                    \
            if (dlogits) launch_rows<TYPE, true, true>(in, out, pol, stream);   \
            else launch_rows<TYPE, true, false>(in, out, pol, stream);          \
        } while (0)
        if (kind == SMLVM_F32) POLICY_ROWS(float);
        else if (kind == SMLVM_F16) POLICY_ROWS(f16_t);
        else POLICY_ROWS(bf16_t);
#undef POLICY_ROWS
    }
    hipLaunchKernelGGL(sum_kernel, dim3(1), dim3(1024), 0, stream, ws + 1, (uint32_t)rows, pol.norm, pol.norm_dev, loss);
    return check_launch();
}
