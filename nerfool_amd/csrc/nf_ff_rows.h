// The gated feed-forward block's products for few rows (new tokens): the weights, read once, are all that counts.
//
// out[m][n] = sum over k of X[m][k] W[n][k], m < 16 NT.  A workgroup owns 16 rows n of the weights (gated: gate and up rows of the same 16 features, in 8 bits of the 32
// features of a block), its waves take turns along k.  A lane loads 16 bytes of a weight row straight into the operand registers of a 16 x 16 matrix
// instruction (A: 16 weight rows, B: 16 tokens): lane l holds row l mod 16, k = V (l / 16) .. + V - 1 of each step, for both operands alike, so that any
// order of k inside a step is right.  A wave keeps two units of 4 (2) steps in flight.  The waves' sums meet in LDS, in the order of the waves.
// Rows may start at any element's address: nothing is padded or copied.
//
// 1 x 4096 x 8192 bf16: gate and up 29 to 32 us, down 14 us (4.2 to 4.8 TB/s; a copy reaches 5.1); 40 x 2048 x 5504 float16: 23 and 17 us, where the tokens' rows, read again by
// every workgroup through the L2, are as many bytes as the weights.
//
// float32 uses the float32 matrix instruction (the weights' bytes bound it up to 32 tokens); 8-bit values become bfloat16 operands, exactly.
#pragma once

#include "nf_ff.h"
#include "nf_ff_sides.h"

template <typename T>
struct FfRow;          // a step: 16 bytes a lane of each operand
template <>
struct FfRow<ff_bf16> {
    typedef FfVec<ff_bf16>::V V;
    static constexpr int KV = 8;          // values a lane and step
    static __device__ __forceinline__ ff_f32x4 mul(V a, V b, ff_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ff_bf16x8, a), __builtin_bit_cast(ff_bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct FfRow<ff_half> {
    typedef FfVec<ff_half>::V V;
    static constexpr int KV = 8;
    static __device__ __forceinline__ ff_f32x4 mul(V a, V b, ff_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ff_half8, a), __builtin_bit_cast(ff_half8, b), c, 0, 0, 0);
    }
};
template <>
struct FfRow<float> {
    typedef FfVec<float>::V V;
    static constexpr int KV = 4;
    static __device__ __forceinline__ ff_f32x4 mul(V a, V b, ff_f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

template <typename T>
__device__ __forceinline__ typename FfRow<T>::V ff_row_load(const T* row, int k, int K) {
    constexpr int KV = FfRow<T>::KV;
    typename FfRow<T>::V v;
    if (k + KV <= K) return *reinterpret_cast<const typename FfRow<T>::V*>(row + k);
#pragma unroll
    for (int j = 0; j < KV; ++j) v[j] = k + j < K ? row[k + j] : (T)0.f;
    return v;
}

// steps of a unit: two units are in flight in registers
constexpr int ff_rows_unit(int nt, bool gated) { return gated && nt == 4 ? 2 : 4; }
// most waves of a workgroup: 64 KB of LDS for their sums, and registers for the two units in flight (and for relu's sides)
constexpr int ff_rows_most(int nt, bool sides) { return nt == 1 && !sides ? 16 : 8; }

// the waves' sums of fragment f: part[wave][f][lane]
__device__ __forceinline__ ff_f32x4 ff_rows_total(const ff_f32x4* part, int waves, int frags, int f, int lane) {
    ff_f32x4 s = part[f * 64 + lane];
    for (int w = 1; w < waves; ++w) s += part[(w * frags + f) * 64 + lane];
    return s;
}

// A wave's units along k: wave, wave + waves, ...  Each workgroup begins at another of them: rows whose length is a power of two lie in the same memory
// channels at the same k, and workgroups that all read the same k at the same time would share a few channels.
struct FfRounds {
    int n, first, stride, unit, base;
    __device__ __forceinline__ FfRounds(int K, int unit_, int waves, int wave, int block) {
        const int units = (K + unit_ - 1) / unit_;
        unit = unit_;
        base = wave * unit_;
        stride = waves * unit_;
        n = wave < units ? (units - wave - 1) / waves + 1 : 0;
        first = n ? block % n : 0;
    }
    __device__ __forceinline__ int at(int i) const {
        int r = first + i;
        if (r >= n) r -= n;
        return base + r * stride;
    }
};

template <typename T, int NT, bool GATED, bool SIDES>
__global__ void __launch_bounds__(64 * ff_rows_most(NT, SIDES)) k_ff_rows(const T* __restrict__ w0, const T* __restrict__ w1, const T* __restrict__ x, int M, int N, int K,
                                                  T* __restrict__ out, float* __restrict__ g_save, float* __restrict__ u_save, int act, FfSides sides) {
    typedef FfRow<T> R;
    typedef typename R::V V;
    constexpr int NW = GATED ? 2 : 1, U = ff_rows_unit(NT, GATED), STEP = 4 * R::KV, UNIT = U * STEP;
    HIP_DYNAMIC_SHARED(ff_f32x4, part)
    const int t0 = blockIdx.y * 16 * NT;          // this workgroup's first token
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, kl = (lane >> 4) * R::KV, n0 = blockIdx.x * 16;
    const int n = n0 + r < N ? n0 + r : N - 1;
    const T* wr[NW];
    wr[0] = w0 + (int64_t)n * K;
    if (GATED) wr[NW - 1] = w1 + (int64_t)n * K;
    const T* xr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xr[t] = x + (int64_t)(t0 + 16 * t + r < M ? t0 + 16 * t + r : M - 1) * K;
    ff_f32x4 acc[NW][NT];
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = ff_f32x4{0.f, 0.f, 0.f, 0.f};
    V a[2][U][NW], b[2][U][NT];
    auto fetch = [&](int s, int k0) {
        if (k0 + UNIT <= K) {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int k = k0 + j * STEP + kl;
#pragma unroll
                for (int i = 0; i < NW; ++i) a[s][j][i] = *reinterpret_cast<const V*>(wr[i] + k);
#pragma unroll
                for (int t = 0; t < NT; ++t) b[s][j][t] = *reinterpret_cast<const V*>(xr[t] + k);
            }
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int k = k0 + j * STEP + kl;
#pragma unroll
                for (int i = 0; i < NW; ++i) a[s][j][i] = ff_row_load(wr[i], k, K);
#pragma unroll
                for (int t = 0; t < NT; ++t) b[s][j][t] = ff_row_load(xr[t], k, K);
            }
        }
    };
    auto multiply = [&](int s) {
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int i = 0; i < NW; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = R::mul(a[s][j][i], b[s][j][t], acc[i][t]);
    };
    const FfRounds o(K, UNIT, waves, wave, blockIdx.x);
    if (o.n > 0) fetch(0, o.at(0));
    for (int i = 0; i < o.n; i += 2) {
        if (i + 1 < o.n) fetch(1, o.at(i + 1));
        multiply(0);
        if (i + 1 >= o.n) break;
        if (i + 2 < o.n) fetch(0, o.at(i + 2));
        multiply(1);
    }
    constexpr int FRAGS = NW * NT;
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[(wave * FRAGS + i * NT + t) * 64 + lane] = acc[i][t];
    __syncthreads();
    for (int t = wave; t < NT; t += waves) {
        const int m = t0 + 16 * t + r, nn = n0 + 4 * (lane >> 4);
        ff_f32x4 v = ff_rows_total(part, waves, FRAGS, t, lane);
        ff_f32x4 u = v;
        if (GATED) u = ff_rows_total(part, waves, FRAGS, (NW - 1) * NT + t, lane);
        if constexpr (SIDES) {          // (as a branch at run time it costs one token 47 -> 50 us)
ff_sides_settle4<T>(sides, m < M && nn < N, m, nn, N - nn, v);
        }
        if (m >= M) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (nn + c >= N) continue;
            const int64_t at = (int64_t)m * N + nn + c;
            float y = v[c];
            if (GATED) {
                float ac, slope;
                ff_act(act, v[c], ac, slope);
                y = ac * u[c];
                if (g_save) {
                    g_save[at] = v[c];
                    u_save[at] = u[c];
                }
            }
            out[at] = (T)y;
        }
    }
}

// waves of a workgroup: as many as fill the chip (2048 waves are 8 a CU), no more than there are units along k, at most `most`
static inline int ff_rows_waves(int groups, int units, int most) {
    int w = 1;
    while (w < most && w < units && groups * w < 2048) w *= 2;
    return w;
}

// Sixteens of tokens a workgroup takes: all of them, as each workgroup reads its weight rows from memory; but where those are too few rows for the CUs, the tokens
// are dealt to several workgroups, and the weights come from the caches for all but one (40 x 2048 from 5504: 20 -> 17 us)
static inline int ff_rows_tokens(int M, int groups) {
    const int all = (M + 15) / 16;
    return groups >= 256 ? all : (all + (256 + groups - 1) / groups - 1) / ((256 + groups - 1) / groups);
}

template <typename T, int NT, bool GATED, bool SIDES>
int ff_rows_launch(const void* w0, const void* w1, const void* x, int M, int N, int K, void* out, float* g_save, float* u_save, int act, const FfSides& sides, hipStream_t st) {
    const int groups = (N + 15) / 16, unit = ff_rows_unit(NT, GATED) * 4 * FfRow<T>::KV;
    const int waves = ff_rows_waves(groups, (K + unit - 1) / unit, ff_rows_most(NT, SIDES));
    hipLaunchKernelGGL((k_ff_rows<T, NT, GATED, SIDES>), dim3(groups, (M + 16 * NT - 1) / (16 * NT)), dim3(64 * waves), (size_t)waves * (GATED ? 2 : 1) * NT * 1024, st, (const T*)w0, (const T*)w1,
                       (const T*)x, M, N, K, (T*)out, g_save, u_save, act, sides);
    return 0;
}
