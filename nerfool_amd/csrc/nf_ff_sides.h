// relu's side of zero for the backward pass.  relu'(g) jumps where g = x . w passes zero: a float32 sum that comes out on the other side of zero than the exact one changes the
// gradient by that unit's whole share, however small |g| is (1500 x 500 x 1333 float32: one unit of two million, and dx is off by 4e-4 of its norm).  So a unit whose |g| does
// not exceed what its float32 sum may be off by is summed again in double, by its whole wave, before g is stored: products of float32 values are exact there, and the sum's own
// error is 2^-29 of the float32 one.
//
// A sum in n additions, cut off or rounded, is off by at most n 2^-23 of its largest partial sum.  Where the whole sum is next to zero its first terms are the negative of its last
// ones, so that no partial sum exceeds |x| |w| / 2 (Cauchy-Schwarz on both ends).  n is the number of matrix instructions behind a sum: D / 32 for 16-bit values, 6 D / 32 for
// float32 in three parts, D / 4 for float32 with few rows.  The bound here is (8 + n) 2^-24 |x| |w|; the 8 takes in the products of parts that are left out (3 2^-24).  Of values like a
// network's that is one unit in some thousand: with all gradients 4096 x 2048 x 8192 bf16 1183 -> 1229 us, 4096 x 4096 x 4096 float32 6389 -> 6584, 1500 x 500 x 1333 float32 189 -> 197
// (row norms and sums), 32768 x 64 x 256 float32 with dx 69 -> 85; activations other than relu have kernels without it.
#pragma once

#include "nf_ff.h"

struct FfSides {
    const void *x, *w;          // [M, D], [F, D], of the kernel's type
    const float *xn, *wn;       // |row|; null: the sides are not asked for
    int D;
    float scale;                // of |x| |w|
};

// N elements of a row from c on, zeros behind its end
template <typename T>
__device__ __forceinline__ typename FfVec<T>::V ff_side_load(const T* row, int c, int dim) {
    constexpr int N = FfVec<T>::N;
    if (c + N <= dim) return *reinterpret_cast<const typename FfVec<T>::V*>(row + c);
    typename FfVec<T>::V v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = c + j < dim ? row[c + j] : (T)0.f;
    return v;
}

// every lane of the wave calls this; `ask`: the lane has a unit (m, n) with the float32 sum g
template <typename T>
__device__ __forceinline__ float ff_side(const FfSides& s, bool ask, int64_t m, int64_t n, float g) {
    constexpr int N = FfVec<T>::N;
    uint64_t todo = __ballot(ask && fabsf(g) <= s.scale * s.xn[ask ? m : 0] * s.wn[ask ? n : 0]);
    const int lane = threadIdx.x & 63;
    while (todo) {
        const int l = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        const T* x = (const T*)s.x + __shfl(m, l, NF_WAVE) * s.D;
        const T* w = (const T*)s.w + __shfl(n, l, NF_WAVE) * s.D;
        double sum = 0;
        constexpr int AHEAD = 4;          // loads under way together: the wave waits for these, not for the sums
        for (int c0 = lane * N; c0 < s.D; c0 += AHEAD * 64 * N) {
            typename FfVec<T>::V a[AHEAD], b[AHEAD];          // (as loaded: converted they would take twice the registers)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                a[i] = ff_side_load(x, c0 + i * 64 * N, s.D);
                b[i] = ff_side_load(w, c0 + i * 64 * N, s.D);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) sum = fma((double)a[i][j], (double)b[i][j], sum);
        }
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) sum += __shfl_xor(sum, k, NF_WAVE);
        if (lane == l) g = (float)sum;
    }
    return g;
}

// |row| of x's M rows, then of w's F: a wave a row
template <typename T>
__global__ void __launch_bounds__(256) k_ff_row_norms(const T* __restrict__ x, int64_t M, const T* __restrict__ w, int64_t F, int D, float* __restrict__ out) {
    constexpr int N = FfVec<T>::N;
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < M + F; r += (int64_t)gridDim.x * 4) {
        const T* row = r < M ? x + r * D : w + (r - M) * D;
        double sq = 0;          // (no square leaves the range)
        for (int c = lane * N; c < D; c += 64 * N) {
            float v[N];
            ff_load_row(row, c, D, v);
#pragma unroll
            for (int j = 0; j < N; ++j) sq = fma((double)v[j], (double)v[j], sq);
        }
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) sq += __shfl_xor(sq, k, NF_WAVE);
        if (lane == 0) out[r] = (float)sqrt(sq);
    }
}

// out: M + F floats; additions: n
template <typename T>
FfSides ff_sides(const void* x, const void* w, int64_t M, int F, int D, int additions, float* out, hipStream_t st) {
    int64_t blocks = (M + F + 3) / 4;
    if (blocks > 2048) blocks = 2048;
    hipLaunchKernelGGL((k_ff_row_norms<T>), dim3((unsigned)blocks), dim3(256), 0, st, (const T*)x, M, (const T*)w, (int64_t)F, D, out);
    return FfSides{x, w, out, out + M, D, ldexpf(8.f + (float)additions, -24)};
}
