// relu's side of zero for the backward pass.  relu'(g) jumps where g = x . w passes zero: a float32 sum that comes out on the other side of zero than the exact one changes the
// gradient by that unit's whole share, however small |g| is (1500 x 500 x 1333 float32: one unit of two million, and dx is off by 4e-4 of its norm).  So a unit whose |g| does
// not exceed what its float32 sum may be off by is summed again in double, by its whole wave, before g is stored: products of float32 values are exact there, and the sum's own
// error is 2^-29 of the float32 one.
//
// A sum in n additions, cut off or rounded, is off by at most n 2^-23 of its largest partial sum.  Where the whole sum is next to zero its first terms are the negative of its last
// ones, so that no partial sum exceeds |x| |w| / 2 (Cauchy-Schwarz on both ends).  n is the number of matrix instructions behind a sum: D / 32 for 16-bit values, 6 D / 32 for
// float32 in three parts, D / 4 for float32 with few rows.  The bound here is (8 + n) 2^-24 |x| |w|; the 8 takes in the products of parts that are left out (3 2^-24).  Of values like a
// network's that is one unit in some thousand: with all gradients 4096 x 2048 x 8192 bf16 1183 -> 1229 us, 4096 x 4096 x 4096 float32 6389 -> 6584, 1500 x 500 x 1333 float32 189 -> 197
// (row norms and sums); the backward kernels of 32768 x 64 x 256, which make the norms beside their own work, float32 37 -> 44, bf16 18 -> 25.  Activations other than relu have
// kernels without it.
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

// the bound of the units of row m, per |w|
__device__ __forceinline__ float ff_side_bound(const FfSides& s, int64_t m) { return s.scale * s.xn[m]; }

// every lane of the wave calls this; the lane has the units (m, n[c]) with the float32 sums g[c], and asks for those within their bound
template <typename T, int COUNT>
__device__ __forceinline__ void ff_sides_settle(const FfSides& s, const bool (&ask)[COUNT], int64_t m, const int (&n)[COUNT], float (&g)[COUNT]) {
    constexpr int N = FfVec<T>::N;
    bool any = false;
#pragma unroll
    for (int c = 0; c < COUNT; ++c) any |= ask[c];
    if (!__ballot(any)) return;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < COUNT; ++c) {
        uint64_t todo = __ballot(ask[c]);
        while (todo) {
            const int l = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            const T* x = (const T*)s.x + __shfl(m, l, NF_WAVE) * s.D;
            const T* w = (const T*)s.w + (int64_t)__shfl(n[c], l, NF_WAVE) * s.D;
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
            if (lane == l) g[c] = (float)sum;
        }
    }
}
// ... n consecutive: n .. n + 3, of which `left` exist
template <typename T>
__device__ __forceinline__ void ff_sides_settle4(const FfSides& s, bool inside, int64_t m, int n, int left, ff_f32x4& g) {
    bool ask[4];
    int at[4];
    float v[4];
    const float bound = inside ? ff_side_bound(s, m) : 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        at[c] = n + c;
        v[c] = g[c];
        ask[c] = inside && c < left;
        ask[c] = ask[c] && fabsf(v[c]) <= bound * s.wn[ask[c] ? n + c : 0];
    }
    ff_sides_settle<T>(s, ask, m, at, v);
    g = ff_f32x4{v[0], v[1], v[2], v[3]};
}

// |row| of x's M rows, then of w's F: LANES lanes a row
template <typename T, int LANES>
__global__ void __launch_bounds__(256) k_ff_row_norms(const T* __restrict__ x, int64_t M, const T* __restrict__ w, int64_t F, int D, float* __restrict__ out) {
    constexpr int N = FfVec<T>::N, ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < M + F; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t r = r0 + threadIdx.x / LANES;
        double sq = 0;          // (no square leaves the range)
        if (r < M + F) {
            const T* row = r < M ? x + r * D : w + (r - M) * D;
            for (int c = lane * N; c < D; c += LANES * N) {
                float v[N];
                ff_load_row(row, c, D, v);
#pragma unroll
                for (int j = 0; j < N; ++j) sq = fma((double)v[j], (double)v[j], sq);
            }
        }
#pragma unroll
        for (int k = LANES / 2; k >= 1; k >>= 1) sq += __shfl_xor(sq, k, NF_WAVE);
        if (r < M + F && lane == 0) out[r] = (float)sqrt(sq);
    }
}

static inline float ff_sides_scale(int additions) { return ldexpf(8.f + (float)additions, -24); }

// out: M + F floats; additions: n
template <typename T>
FfSides ff_sides(const void* x, const void* w, int64_t M, int F, int D, int additions, float* out, hipStream_t st) {
    const auto run = [&](auto kernel, int lanes) {
        int64_t blocks = (M + F + 256 / lanes - 1) / (256 / lanes);
        if (blocks > 2048) blocks = 2048;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, (const T*)x, M, (const T*)w, (int64_t)F, D, out);
    };
    if (D <= 16 * FfVec<T>::N) run(k_ff_row_norms<T, 16>, 16);
    else run(k_ff_row_norms<T, 64>, 64);
    return FfSides{x, w, out, out + M, D, ff_sides_scale(additions)};
}
