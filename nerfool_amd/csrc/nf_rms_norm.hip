// Root-mean-square norm with the residual's addition, forward and backward, and rows brought to 8 bits with block scales -- what stands in
// front of a feed-forward block (gnt/transformer_network.py:121-171 norms with LayerNorm before its feed-forward; this is the form without a mean).
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = w h rstd
//   dx = dr = rstd (w dy - xhat mean(w dy xhat)) + dh,  dw = sum over rows of dy xhat,  xhat = h rstd
//
// HBM bounds it: every tensor is read or written once.  A row's values stay in registers between the statistics and their use; a row is
// owned by 8 to 64 lanes of a wave or, above 64 (128 where there are many rows) vectors of 16 bytes, by a workgroup; rows longer than 4096 vectors are
// read twice.  The squares and sums are float; y is made from the float sum x + r, not from h as rounded.
// 8192 x 4096 bf16 with a residual to 8 bits: 49 us, 4.8 TB/s of the 5.1 that a copy reaches; 32768 x 64 float32: forward 8.6 us, backward 8.9 + 2.4 us for dw's
// partial sums; one row of 4096: 3.2 us, a launch.
#include "nf_ff.h"

namespace {

struct RmsArgs {
    const void *x, *r, *w;
    void *h, *y;
    uint8_t *q, *s;
    float* rstd;
    int64_t rows;
    int dim;
    float eps;
};

// sum over the TPR threads of a row; TPR <= 64: a butterfly inside the wave, else over the waves of the workgroup (`part`: one float a wave)
template <int TPR, typename A>
__device__ __forceinline__ A rms_row_sum(A v, A* part) {
#pragma unroll
    for (int m = (TPR < 64 ? TPR : 64) / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, NF_WAVE);
    if (TPR > 64) {
        __syncthreads();          // the previous row's sums have been read
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += part[i];
    }
    return v;
}

// v: N values of a row in block `c / 32`; the 32 / N lanes that hold a block reduce its maximum
template <int N>
__device__ __forceinline__ void rms_store_8bit(uint8_t* q, uint8_t* s, int c, int dim, const float* v) {
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        top = fmaxf(top, fabsf(v[j]));
        bad |= !(fabsf(v[j]) <= 3.4028235e38f);
    }
    if (bad) top = INFINITY;          // fmaxf drops a NaN
    top = nf_grp_reduce<32 / N>(top, NfMax());
    const unsigned byte = ff_scale_byte(top);
    if (c >= dim) return;
    const float inv = byte == 255u ? NAN : ff_scale_inverse(byte);
    unsigned u[N / 4];
#pragma unroll
    for (int g = 0; g < N / 4; ++g) u[g] = ff_e4m3x4(v[4 * g] * inv, v[4 * g + 1] * inv, v[4 * g + 2] * inv, v[4 * g + 3] * inv);
    if (c % 32 == 0) s[c / 32] = (uint8_t)byte;
    if (c + N <= dim) {
        typedef unsigned U __attribute__((ext_vector_type(N / 4 > 1 ? 2 : 1), aligned(1)));
        U t;
#pragma unroll
        for (int g = 0; g < N / 4; ++g) t[g] = u[g];
        *reinterpret_cast<U*>(q + c) = t;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < dim) q[c + j] = (uint8_t)(u[j / 4] >> (8 * (j % 4)));
    }
}

// y of an 8-bit row is made in double, of the float sums x + r: a value next to a border of the grid takes the neighbouring step for an error of
// one part in 2^24, and beside the memory's time the doubles cost nothing
template <int MODE>
struct RmsAcc {
    typedef float A;
};
template <>
struct RmsAcc<1> {
    typedef double A;
};

enum { RMS_SAME = 0, RMS_8BIT = 1, RMS_QUANT = 2 };          // y in the inputs' type; y in 8 bits; x itself in 8 bits

template <typename T, int TPR, int NV, int MODE>
__global__ void __launch_bounds__(TPR <= 256 ? 256 : TPR) k_rms_fwd(RmsArgs a) {
    typedef typename RmsAcc<MODE>::A A;
    constexpr int N = FfVec<T>::N, BLOCK = TPR <= 256 ? 256 : TPR, RPB = TPR <= 64 ? BLOCK / TPR : 1;
    __shared__ A part[16];
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, sub = TPR <= 64 ? threadIdx.x / TPR : 0;
    const int dim = a.dim;
    float w[NV][N];
    if (MODE != RMS_QUANT) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (a.w)
                ff_load_row((const T*)a.w, (j * TPR + t) * N, dim, w[j]);
            else
                for (int i = 0; i < N; ++i) w[j][i] = 1.f;
        }
    }
    // every thread of a workgroup makes the same number of rounds: the sums are collective
    for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = row0 + sub;
        const bool live = row < a.rows;
        const int64_t at = (live ? row : a.rows - 1) * dim;
        float v[NV][N];
        A sq = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            ff_load_row((const T*)a.x + at, (j * TPR + t) * N, dim, v[j]);
            if (MODE != RMS_QUANT && a.r) {
                float r[N];
                ff_load_row((const T*)a.r + at, (j * TPR + t) * N, dim, r);
#pragma unroll
                for (int i = 0; i < N; ++i) v[j][i] += r[i];
            }
        }
        if (MODE != RMS_QUANT) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) sq = fma((A)v[j][i], (A)v[j][i], sq);
            sq = rms_row_sum<TPR>(sq, part);
            const A rstd = (A)1 / sqrt(sq / (A)dim + (A)a.eps);
            if (a.rstd && t == 0 && live) a.rstd[row] = (float)rstd;
            if (a.h && live) {
#pragma unroll
                for (int j = 0; j < NV; ++j) ff_store_row((T*)a.h + at, (j * TPR + t) * N, dim, v[j]);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) v[j][i] = (float)((A)v[j][i] * rstd * (A)w[j][i]);
        }
        if (MODE == RMS_SAME) {
            if (live) {
#pragma unroll
                for (int j = 0; j < NV; ++j) ff_store_row((T*)a.y + at, (j * TPR + t) * N, dim, v[j]);
            }
        } else {
            const int64_t blocks = (dim + 31) / 32;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                rms_store_8bit<N>(a.q + at, a.s + (live ? row : a.rows - 1) * blocks, (j * TPR + t) * N, live ? dim : 0, v[j]);
        }
    }
}

// rows of any length, read twice: a workgroup per row
template <typename T, int MODE>
__global__ void __launch_bounds__(1024) k_rms_fwd_long(RmsArgs a) {
    typedef typename RmsAcc<MODE>::A A;
    constexpr int N = FfVec<T>::N, STEP = 1024 * N;
    __shared__ A part[16];
    const int dim = a.dim;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * dim;
        float v[N], r[N], w[N];
        A rstd = 1;
        if (MODE != RMS_QUANT) {
            A sq = 0;
            for (int c = threadIdx.x * N; c < dim; c += STEP) {
                ff_load_row((const T*)a.x + at, c, dim, v);
                if (a.r) {
                    ff_load_row((const T*)a.r + at, c, dim, r);
                    for (int i = 0; i < N; ++i) v[i] += r[i];
                }
                for (int i = 0; i < N; ++i) sq = fma((A)v[i], (A)v[i], sq);
                if (a.h) ff_store_row((T*)a.h + at, c, dim, v);
            }
            sq = rms_row_sum<1024>(sq, part);
            rstd = (A)1 / sqrt(sq / (A)dim + (A)a.eps);
            if (a.rstd && threadIdx.x == 0) a.rstd[row] = (float)rstd;
        }
        for (int c0 = 0; c0 < dim; c0 += STEP) {          // every lane stays for the block maxima
            const int c = c0 + threadIdx.x * N;
            ff_load_row((const T*)a.x + at, c, dim, v);
            if (MODE != RMS_QUANT) {
                if (a.r) {
                    ff_load_row((const T*)a.r + at, c, dim, r);
                    for (int i = 0; i < N; ++i) v[i] += r[i];
                }
                for (int i = 0; i < N; ++i) w[i] = 1.f;
                if (a.w) ff_load_row((const T*)a.w, c, dim, w);
                for (int i = 0; i < N; ++i) v[i] = (float)((A)v[i] * rstd * (A)w[i]);
            }
            if (MODE == RMS_SAME)
                ff_store_row((T*)a.y + at, c, dim, v);
            else
                rms_store_8bit<N>(a.q + at, a.s + row * ((dim + 31) / 32), c, dim, v);
        }
    }
}

struct RmsBwdArgs {
    const void *dy, *dh, *h, *r, *w;          // r: nullable, added to h
    const float* rstd;
    void* dx;
    float* partial;          // [gridDim.x][dim], nullable (dw not asked for)
    int64_t rows;
    int dim;
};

// h's values, or x + r
template <typename T>
__device__ __forceinline__ void rms_load_h(const RmsBwdArgs& a, int64_t at, int c, float* v) {
    ff_load_row((const T*)a.h + at, c, a.dim, v);
    if (a.r) {
        float r[FfVec<T>::N];
        ff_load_row((const T*)a.r + at, c, a.dim, r);
#pragma unroll
        for (int i = 0; i < FfVec<T>::N; ++i) v[i] += r[i];
    }
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR <= 256 ? 256 : TPR) k_rms_bwd(RmsBwdArgs a) {
    constexpr int N = FfVec<T>::N, BLOCK = TPR <= 256 ? 256 : TPR, RPB = TPR <= 64 ? BLOCK / TPR : 1;
    __shared__ float part[16];
    __shared__ float sums[TPR <= 64 ? BLOCK * N : 1];
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, sub = TPR <= 64 ? threadIdx.x / TPR : 0;
    const int dim = a.dim;
    float w[NV][N], dw[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (a.w)
            ff_load_row((const T*)a.w, (j * TPR + t) * N, dim, w[j]);
        else
            for (int i = 0; i < N; ++i) w[j][i] = 1.f;
        for (int i = 0; i < N; ++i) dw[j][i] = 0.f;
    }
    for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = row0 + sub;
        const bool live = row < a.rows;
        const int64_t at = (live ? row : a.rows - 1) * dim;
        const float rstd = a.rstd[live ? row : a.rows - 1];
        float g[NV][N], xh[NV][N];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            ff_load_row((const T*)a.dy + at, (j * TPR + t) * N, dim, g[j]);
            rms_load_h<T>(a, at, (j * TPR + t) * N, xh[j]);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                xh[j][i] *= rstd;
                if (live) dw[j][i] = fmaf(g[j][i], xh[j][i], dw[j][i]);
                g[j][i] *= w[j][i];
                dot = fmaf(g[j][i], xh[j][i], dot);
            }
        dot = rms_row_sum<TPR>(dot, part) / (float)dim;
        if (!live) continue;          // (only where a row is a part of a wave: no workgroup barrier follows in the loop)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = 0.f;
            if (a.dh) ff_load_row((const T*)a.dh + at, (j * TPR + t) * N, dim, d);
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = fmaf(rstd, g[j][i] - xh[j][i] * dot, d[i]);
            ff_store_row((T*)a.dx + at, (j * TPR + t) * N, dim, d);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (int64_t)blockIdx.x * dim;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * N;
        if (TPR <= 64) {          // the workgroup's row groups, added in their order
            __syncthreads();
            for (int i = 0; i < N; ++i) sums[threadIdx.x * N + i] = dw[j][i];
            __syncthreads();
            if (sub == 0)
                for (int i = 0; i < N; ++i) {
                    float s = 0.f;
                    for (int k = 0; k < RPB; ++k) s += sums[(k * TPR + t) * N + i];
                    dw[j][i] = s;
                }
        }
        if (sub == 0)
            for (int i = 0; i < N; ++i)
                if (c + i < dim) out[c + i] = dw[j][i];
    }
}

// dx of rows of any length, read twice
template <typename T>
__global__ void __launch_bounds__(1024) k_rms_bwd_long(RmsBwdArgs a) {
    constexpr int N = FfVec<T>::N, STEP = 1024 * N;
    __shared__ float part[16];
    const int dim = a.dim;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * dim;
        const float rstd = a.rstd[row];
        float g[N], xh[N], w[N], d[N], dot = 0.f;
        for (int c = threadIdx.x * N; c < dim; c += STEP) {
            for (int i = 0; i < N; ++i) w[i] = 1.f;
            if (a.w) ff_load_row((const T*)a.w, c, dim, w);
            ff_load_row((const T*)a.dy + at, c, dim, g);
            rms_load_h<T>(a, at, c, xh);
            for (int i = 0; i < N; ++i) dot = fmaf(g[i] * w[i], xh[i] * rstd, dot);
        }
        dot = rms_row_sum<1024>(dot, part) / (float)dim;
        for (int c = threadIdx.x * N; c < dim; c += STEP) {
            for (int i = 0; i < N; ++i) w[i] = 1.f, d[i] = 0.f;
            if (a.w) ff_load_row((const T*)a.w, c, dim, w);
            if (a.dh) ff_load_row((const T*)a.dh + at, c, dim, d);
            ff_load_row((const T*)a.dy + at, c, dim, g);
            rms_load_h<T>(a, at, c, xh);
            for (int i = 0; i < N; ++i) d[i] = fmaf(rstd, g[i] * w[i] - xh[i] * rstd * dot, d[i]);
            ff_store_row((T*)a.dx + at, c, dim, d);
        }
    }
}
// ... and their dw: a thread per column and slice of the rows -> partial[slice][dim]
template <typename T>
__global__ void __launch_bounds__(256) k_rms_dw_long(RmsBwdArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.dim) return;
    float s = 0.f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
        s = fmaf((float)((const T*)a.dy)[row * a.dim + c], ((float)((const T*)a.h)[row * a.dim + c] + (a.r ? (float)((const T*)a.r)[row * a.dim + c] : 0.f)) * a.rstd[row], s);
    a.partial[(int64_t)blockIdx.y * a.dim + c] = s;
}

// dw[c] = sum of the n partial sums, in a fixed order: 32 columns x 32 slices a workgroup
template <typename T>
__global__ void __launch_bounds__(1024) k_rms_dw(const float* __restrict__ partial, int n, int dim, T* __restrict__ dw) {
    __shared__ float sums[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    float s = 0.f;
    if (c < dim) {
#pragma unroll 8
        for (int i = slice; i < n; i += 32) s += partial[(int64_t)i * dim + c];
    }
    sums[slice][col] = s;
    __syncthreads();
    if (slice == 0 && c < dim) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sums[i][col];
        dw[c] = (T)s;
    }
}

constexpr int RMS_MAX_PARTIALS = 512;

int64_t rms_grid(int64_t rows, int rows_per_block, int64_t most) {
    int64_t g = (rows + rows_per_block - 1) / rows_per_block;
    return g < most ? g : most;
}

// vectors of 16 bytes in a row -> threads a row and vectors a thread.  Up to 64 vectors the row is a part of a wave; up to 128 a wave owns it where there are 2048 rows
// or more (8 waves a CU; the sums need no barrier), else, and above, a workgroup does: of 512 vectors a wave holds 240 registers and reads 8192 rows in 138 us,
// a workgroup of four waves in 48.  The border of 2048 rows, of 125 vectors in bf16, us with a workgroup and a wave a row: forward 1024 rows 4.4 and 4.7, 1536 rows 5.1 and 5.1, 2048
// rows 5.9 and 5.4, 8192 rows 14.5 and 11.7; backward 512 rows 8.7 and 8.6, 1024 rows 9.9 and 8.6, 2048 rows 12.2 and 10.2, 8192 rows 31.8 and 19.1.
#define RMS_DISPATCH(VECS, ROWS, GO, LONG)          \
    do {                                            \
        const int nv_ = (VECS);                     \
        const bool many_ = (ROWS) >= 2048;          \
        if (nv_ <= 8) { GO(8, 1); }                 \
        else if (nv_ <= 16) { GO(16, 1); }          \
        else if (nv_ <= 32) { GO(32, 1); }          \
        else if (nv_ <= 64) { GO(64, 1); }          \
        else if (many_ && nv_ <= 128) { GO(64, 2); }\
        else if (nv_ <= 256) { GO(256, 1); }        \
        else if (nv_ <= 512) { GO(256, 2); }        \
        else if (nv_ <= 1024) { GO(256, 4); }       \
        else if (nv_ <= 2048) { GO(512, 4); }       \
        else if (nv_ <= 4096) { GO(1024, 4); }      \
        else { LONG; }                              \
    } while (0)

template <typename T, int MODE>
void rms_fwd(const RmsArgs& a, hipStream_t st) {
    const int64_t most = 256 * 8;
#define GO(TPR, NV)                                                                                                                  \
    hipLaunchKernelGGL((k_rms_fwd<T, TPR, NV, MODE>), dim3((unsigned)rms_grid(a.rows, TPR <= 64 ? 256 / TPR : 1, most)), \
                       dim3(TPR <= 256 ? 256 : TPR), 0, st, a)
    RMS_DISPATCH((a.dim + FfVec<T>::N - 1) / FfVec<T>::N, a.rows, GO,
                 hipLaunchKernelGGL((k_rms_fwd_long<T, MODE>), dim3((unsigned)rms_grid(a.rows, 1, 512)), dim3(1024), 0, st, a));
#undef GO
}

template <typename T>
void rms_bwd(const RmsBwdArgs& a, void* dw, hipStream_t st) {
    int n = 0;
#define GO(TPR, NV)                                                                                                        \
    n = (int)rms_grid(a.rows, TPR <= 64 ? 256 / TPR : 1, a.partial ? RMS_MAX_PARTIALS : 2048);                             \
    hipLaunchKernelGGL((k_rms_bwd<T, TPR, NV>), dim3((unsigned)n), dim3(TPR <= 256 ? 256 : TPR), 0, st, a)
    RMS_DISPATCH((a.dim + FfVec<T>::N - 1) / FfVec<T>::N, a.rows, GO, {
        hipLaunchKernelGGL((k_rms_bwd_long<T>), dim3((unsigned)rms_grid(a.rows, 1, 512)), dim3(1024), 0, st, a);
        if (a.partial) {
            n = (int)rms_grid(a.rows, 1, 32);
            hipLaunchKernelGGL((k_rms_dw_long<T>), dim3((a.dim + 255) / 256, n), dim3(256), 0, st, a);
        }
    });
#undef GO
    if (a.partial) hipLaunchKernelGGL((k_rms_dw<T>), dim3((a.dim + 31) / 32), dim3(1024), 0, st, (const float*)a.partial, n, a.dim, (T*)dw);
}

}  // namespace

extern "C" int nf_rms_norm_fwd(const void* x, const void* residual, const void* weight, int64_t rows, int dim, int dtype, float eps, void* h,
                               void* y, uint8_t* q, uint8_t* scale, float* rstd, nf_stream_t stream) {
    NF_REQUIRE(rows >= 0 && dim >= 1 && dim <= (1 << 24) && dtype >= FF_F32 && dtype <= FF_F16,
               "nf_rms_norm_fwd: need rows >= 0, 1 <= dim <= 2^24, dtype in 0 .. 2 (got rows %lld dim %d dtype %d)", (long long)rows, dim, dtype);
    NF_REQUIRE((y != nullptr) != (q != nullptr) && (q != nullptr) == (scale != nullptr),
               "nf_rms_norm_fwd: either y, or q and scale");
    NF_REQUIRE(!residual || h, "nf_rms_norm_fwd: a residual needs h, where the sum goes");
    if (rows == 0) return 0;
    const RmsArgs a = {x, residual, weight, residual ? h : nullptr, y, q, scale, rstd, rows, dim, eps};
    hipStream_t st = (hipStream_t)stream;
    if (y) {
        if (dtype == FF_F32) rms_fwd<float, RMS_SAME>(a, st);
        else if (dtype == FF_BF16) rms_fwd<ff_bf16, RMS_SAME>(a, st);
        else rms_fwd<ff_half, RMS_SAME>(a, st);
    } else {
        if (dtype == FF_F32) rms_fwd<float, RMS_8BIT>(a, st);
        else if (dtype == FF_BF16) rms_fwd<ff_bf16, RMS_8BIT>(a, st);
        else rms_fwd<ff_half, RMS_8BIT>(a, st);
    }
    NF_LAUNCH_CHECK("nf_rms_norm_fwd");
    return 0;
}

extern "C" int64_t nf_rms_norm_bwd_workspace_floats(int dim) { return (int64_t)RMS_MAX_PARTIALS * dim; }

extern "C" int nf_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* residual, const void* weight, const float* rstd, int64_t rows, int dim,
                               int dtype, void* dx, void* dweight, float* workspace, nf_stream_t stream) {
    NF_REQUIRE(rows >= 1 && dim >= 1 && dim <= (1 << 24) && dtype >= FF_F32 && dtype <= FF_F16,
               "nf_rms_norm_bwd: need rows >= 1, 1 <= dim <= 2^24, dtype in 0 .. 2 (got rows %lld dim %d dtype %d)", (long long)rows, dim, dtype);
    NF_REQUIRE(!dweight || workspace, "nf_rms_norm_bwd: dweight needs a workspace");
    const RmsBwdArgs a = {dy, dh, h, residual, weight, rstd, dx, dweight ? workspace : nullptr, rows, dim};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FF_F32) rms_bwd<float>(a, dweight, st);
    else if (dtype == FF_BF16) rms_bwd<ff_bf16>(a, dweight, st);
    else rms_bwd<ff_half>(a, dweight, st);
    NF_LAUNCH_CHECK("nf_rms_norm_bwd");
    return 0;
}

extern "C" int nf_quantize_8bit(const void* x, int64_t rows, int dim, int dtype, uint8_t* q, uint8_t* scale, nf_stream_t stream) {
    NF_REQUIRE(rows >= 0 && dim >= 1 && dim <= (1 << 24) && dtype >= FF_F32 && dtype <= FF_F16,
               "nf_quantize_8bit: need rows >= 0, 1 <= dim <= 2^24, dtype in 0 .. 2 (got rows %lld dim %d dtype %d)", (long long)rows, dim, dtype);
    if (rows == 0) return 0;
    const RmsArgs a = {x, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, dim, 0.f};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FF_F32) rms_fwd<float, RMS_QUANT>(a, st);
    else if (dtype == FF_BF16) rms_fwd<ff_bf16, RMS_QUANT>(a, st);
    else rms_fwd<ff_half, RMS_QUANT>(a, st);
    NF_LAUNCH_CHECK("nf_quantize_8bit");
    return 0;
}
