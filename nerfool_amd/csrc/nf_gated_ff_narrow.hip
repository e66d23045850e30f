// The gated feed-forward block at the widths of the ray transformer (dim <= 64: gnt/transformer_network.py:38-50 has 64 and 256) in one kernel a direction: what the block
// computes between its input and its output never leaves the registers.
//
// A wave owns 16 tokens.  The features are walked in chunks of 32: g and u of the chunk are made as 16 x 16 blocks (weights the A operand, tokens the B operand, so that a
// lane holds 4 consecutive features of one token), h of the chunk goes back into B operands as it lies -- the lane's 4 features of the first block are its k 0 .. 3 and those of
// the second its k 4 .. 7; the down projection's records have their features in that order -- and out grows by the chunk's share.  The backward pass to x alone (constant
// weights, as in an attack) makes g and u again instead of reading them: dx += dg Wg + du Wu the same way, with dh = dy Wd of the chunk between.
// The weights come as records of operand fragments (k_ff_narrow_pack, per call), 1 KB each, by LDS-DMA, one chunk ahead, for the eight waves of a workgroup.  float32: three bf16
// parts of every operand, six products (nf_gated_ff.hip); h, dg and du are then split, not rounded.  Bound by the matrix instructions and, as much, by the vector
// instructions of activation and split between them: 32768 x 64 x 256 float32 takes 30 us forward and 43
// backward, and 5 each for the records (in separate products: 69 and 80; four waves of 32 tokens, one a SIMD: 47 and 67).
#include "nf_ff_gemm.h"
#include "nf_ff_sides.h"

namespace {

// ---- records.  A chunk's fragments, KD = padded dim / 32:  gate [2][KD], up [2][KD]; forward: down [2 KD]; backward: down transposed [2][KD], gate and up transposed [2 KD] each
constexpr int narrow_records(int kd, bool backward) { return (backward ? 10 : 6) * kd; }

template <typename T>
struct NarrowParts {
    typedef T E;
    static constexpr int NP = 1;
    static __device__ __forceinline__ void split(float v, E* p) { p[0] = (E)v; }
};
template <>
struct NarrowParts<float> {
    typedef ff_bf16 E;
    static constexpr int NP = 3;
    static __device__ __forceinline__ void split(float v, E* p) { ff_split3(v, p); }
};

// one wave a record: lane l holds row l mod 16, k = 8 (l / 16) + j, j = 0 .. 7 -> [chunk][record][part][lane][8]
template <typename T>
__global__ void __launch_bounds__(256) k_ff_narrow_pack(const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ wd, int D, int F, int kd, int backward,
                                                        typename NarrowParts<T>::E* __restrict__ out, float* __restrict__ norms) {
    typedef NarrowParts<T> P;
    const int per = narrow_records(kd, backward), chunks = (F + 31) / 32;
    const int rec = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, row = lane & 15, q = lane >> 4;
    if (rec >= per * chunks) {          // behind the records: a wave per gate row, whose norm relu's sides ask for
        const int f = rec - per * chunks;
        if (!norms || f >= 32 * chunks) return;
        const double v = f < F && lane < D ? (double)(float)wg[(int64_t)f * D + lane] : 0.0;
        double sq = v * v;
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) sq += __shfl_xor(sq, k, NF_WAVE);
        if (lane == 0) norms[f] = (float)sqrt(sq);
        return;
    }
    const int chunk = rec / per, n = rec - chunk * per;
    typename P::E part[8][P::NP];
    for (int j = 0; j < 8; ++j) {
        const int k = 8 * q + j, f_of_k = 32 * chunk + (j < 4 ? 4 * q + j : 16 + 4 * q + j - 4);
        float v = 0.f;
        if (n < 4 * kd) {                       // gate, up: rows are features, k is dim
            const int i = n % (2 * kd), f = 32 * chunk + 16 * (i / kd) + row, d = 32 * (i % kd) + k;
            if (f < F && d < D) v = (float)(n < 2 * kd ? wg : wu)[(int64_t)f * D + d];
        } else if (!backward) {                 // down: rows are dim, k is features
            const int d = 16 * (n - 4 * kd) + row;
            if (d < D && f_of_k < F) v = (float)wd[(int64_t)d * F + f_of_k];
        } else if (n < 6 * kd) {                // down transposed: rows are features, k is dim
            const int i = n - 4 * kd, f = 32 * chunk + 16 * (i / kd) + row, d = 32 * (i % kd) + k;
            if (f < F && d < D) v = (float)wd[(int64_t)d * F + f];
        } else {                                // gate, up transposed: rows are dim, k is features
            const int i = n - 6 * kd, d = 16 * (i % (2 * kd)) + row;
            if (d < D && f_of_k < F) v = (float)(i < 2 * kd ? wg : wu)[(int64_t)f_of_k * D + d];
        }
        P::split(v, part[j]);
    }
    for (int e = 0; e < P::NP; ++e) {
        typename P::E* o = out + ((int64_t)(rec * P::NP + e) * 64 + lane) * 8;
        for (int j = 0; j < 8; ++j) o[j] = part[j][e];
    }
}

template <typename T, int KD, bool BWD>
struct Narrow {
    typedef NarrowParts<T> P;
    typedef typename P::E E;
    typedef FfMfma<E> Mfma;
    typedef typename Mfma::V V;
    static constexpr int NP = P::NP, RECORDS = narrow_records(KD, BWD), PIECES = RECORDS * NP, CHUNK = PIECES * 1024;

    // this lane's 8 values of a token's row as an operand: k = 32 kd + 8 (l / 16) ..
    static __device__ __forceinline__ void row(const T* x, int64_t m, int64_t M, int D, int k, V (&v)[NP], double* squares = nullptr) {
        float f[8];
        const T* r = x + (m < M ? m : M - 1) * D;
        constexpr int N = FfVec<T>::N;
#pragma unroll
        for (int c = 0; c < 8; c += N) {
            float t[N];
            ff_load_row(r, k + c, D, t);
#pragma unroll
            for (int j = 0; j < N; ++j) f[c + j] = t[j];
        }
        if (squares) {
#pragma unroll
            for (int j = 0; j < 8; ++j) *squares = fma((double)f[j], (double)f[j], *squares);
        }
        operand(f, v);
    }
    static __device__ __forceinline__ void operand(const float (&f)[8], V (&v)[NP]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            E p[NP];
            P::split(f[j], p);
#pragma unroll
            for (int e = 0; e < NP; ++e) v[e][j] = p[e];
        }
    }
    // c += record n x b, smallest products first
    static __device__ __forceinline__ void multiply(const char* lds, int n, int lane, const V (&b)[NP], ff_f32x4& c) {
        V a[NP];
#pragma unroll
        for (int e = 0; e < NP; ++e) a[e] = *reinterpret_cast<const V*>(lds + (n * NP + e) * 1024 + lane * 16);
#pragma unroll
        for (int o = NP - 1; o >= 0; --o)
#pragma unroll
            for (int e = 0; e <= o; ++e) c = Mfma::mul(a[e], b[o - e], c);
    }
};

template <typename T, int KD, bool BWD, bool SIDES>
__global__ void __launch_bounds__(512) k_ff_narrow(const T* __restrict__ x, const T* __restrict__ dy, const char* __restrict__ records, int64_t M, int D, int F, int act,
                                                   T* __restrict__ out, FfSides sides) {
    typedef Narrow<T, KD, BWD> N;
    typedef typename N::V V;
    constexpr int NP = N::NP, WAVES = 8;
    HIP_DYNAMIC_SHARED(char, lds)
    const int lane = threadIdx.x & 63, wave = ff_wave_index(), q = lane >> 4;
    const int64_t m = (int64_t)blockIdx.x * (16 * WAVES) + wave * 16 + (lane & 15);          // this lane's token
    auto load_chunk = [&](int c) {
        const char* src = records + (int64_t)c * N::CHUNK;
        for (int p = wave; p < N::PIECES; p += WAVES) ff_dma16(src + p * 1024, (unsigned)lane * 16, lds, (c & 1) * N::CHUNK + p * 1024, lane);
    };
    load_chunk(0);
    V xb[KD][NP], yb[BWD ? KD : 1][NP];
    double squares = 0;
#pragma unroll
    for (int k = 0; k < KD; ++k) {
        N::row(x, m, M, D, 32 * k + 8 * q, xb[k], SIDES ? &squares : nullptr);
        if (BWD) N::row(dy, m, M, D, 32 * k + 8 * q, yb[BWD ? k : 0]);
    }
    float bound = 0.f;          // of the token's units, per |row of Wg|; the token lies on 4 lanes
    if constexpr (SIDES) {
        squares += __shfl_xor(squares, 16, NF_WAVE);
        squares += __shfl_xor(squares, 32, NF_WAVE);
        bound = sides.scale * (float)sqrt(squares);
    }
    float scale = 1.f;          // float16: of the token's dg and du (ff_grad_scale; its dy lies on 4 lanes)
    if constexpr (BWD && std::is_same<T, ff_half>::value) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)yb[k][0][j]));
        top = fmaxf(top, __shfl_xor(top, 16, NF_WAVE));
        top = fmaxf(top, __shfl_xor(top, 32, NF_WAVE));
        scale = ff_grad_scale(top);
    }
    const int chunks = (F + 31) / 32;
    const ff_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    ff_f32x4 sum[2 * KD];
#pragma unroll
    for (int i = 0; i < 2 * KD; ++i) sum[i] = zero;
    for (int c = 0; c < chunks; ++c) {
        ff_dma_barrier<0>();          // the chunk has landed for every wave, and the other buffer has been read by every wave
        if (c + 1 < chunks) load_chunk(c + 1);
        const char* w = lds + (c & 1) * N::CHUNK;
        ff_f32x4 g[2], u[2], dh[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            g[i] = u[i] = dh[i] = zero;
#pragma unroll
            for (int k = 0; k < KD; ++k) {
                N::multiply(w, i * KD + k, lane, xb[k], g[i]);
                N::multiply(w, (2 + i) * KD + k, lane, xb[k], u[i]);
                if (BWD) N::multiply(w, (4 + i) * KD + k, lane, yb[BWD ? k : 0], dh[i]);
            }
        }
        if constexpr (SIDES) {
            bool ask[8];
            int f[8];
            float gs[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const ff_f32x4 wn = *reinterpret_cast<const ff_f32x4*>(sides.wn + 32 * c + 16 * i + 4 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[4 * i + j] = 32 * c + 16 * i + 4 * q + j;
                    gs[4 * i + j] = g[i][j];
                    ask[4 * i + j] = m < M && f[4 * i + j] < F && fabsf(g[i][j]) <= bound * wn[j];
                }
            }
            ff_sides_settle<T>(sides, ask, m, f, gs);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j / 4][j % 4] = gs[j];
        }
        V hb[NP], ub[NP];          // forward: h; backward: dg and du
        float v[8], v2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gv = g[j / 4][j % 4], uv = u[j / 4][j % 4];
            float a, slope;
            ff_act(act, gv, a, slope);
            if (BWD) {
                const float d = dh[j / 4][j % 4];
                v[j] = d * uv * slope;
                v2[j] = d * a;
                if (std::is_same<T, ff_half>::value) v[j] *= scale, v2[j] *= scale;
            } else
                v[j] = a * uv;
        }
        N::operand(v, hb);
        if (BWD) N::operand(v2, ub);
#pragma unroll
        for (int i = 0; i < 2 * KD; ++i) {
            N::multiply(w, (BWD ? 6 : 4) * KD + i, lane, hb, sum[i]);
            if (BWD) N::multiply(w, 8 * KD + i, lane, ub, sum[i]);
        }
    }
    ff_dma_barrier<0>();          // no load may land in LDS that the workgroup has given back
    if (m >= M) return;
#pragma unroll
    for (int i = 0; i < 2 * KD; ++i) {
        if (BWD && std::is_same<T, ff_half>::value) sum[i] *= 1.f / scale;
        ff_put(out + m * D + 16 * i + 4 * q, D - (16 * i + 4 * q), sum[i]);
    }
}

template <typename T, int KD, bool BWD, bool SIDES>
int narrow_run(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, int64_t M, int D, int F, int act, void* out, void* workspace, hipStream_t st) {
    typedef Narrow<T, KD, BWD> N;
    constexpr int LDS = 2 * N::CHUNK;
    static bool set[NF_MAX_DEVICES];
    const int dev = nf_current_device();
    if (!set[dev]) {
        const hipError_t e = hipFuncSetAttribute((const void*)k_ff_narrow<T, KD, BWD, SIDES>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            nf_set_error("gated feed-forward: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
            return 2;
        }
        set[dev] = true;
    }
    const int chunks = (F + 31) / 32, records = N::RECORDS * chunks;
    float* norms = SIDES ? (float*)((char*)workspace + (int64_t)records * N::NP * 1024) : nullptr;
    const FfSides sides = {x, wg, nullptr, norms, D, ff_sides_scale(N::NP == 3 ? 12 : 2)};
    hipLaunchKernelGGL((k_ff_narrow_pack<T>), dim3((records + (SIDES ? 32 * chunks : 0) + 3) / 4), dim3(256), 0, st, (const T*)wg, (const T*)wu, (const T*)wd, D, F, KD, (int)BWD,
                       (typename N::E*)workspace, norms);
    hipLaunchKernelGGL((k_ff_narrow<T, KD, BWD, SIDES>), dim3((unsigned)((M + 127) / 128)), dim3(512), LDS, st, (const T*)x, (const T*)dy, (const char*)workspace, M, D, F, act,
                       (T*)out, sides);
    return 0;
}
template <typename T, int KD>
int narrow_way(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, int64_t M, int D, int F, int act, void* out, void* workspace, hipStream_t st) {
    if (!dy) return narrow_run<T, KD, false, false>(x, wg, wu, wd, dy, M, D, F, act, out, workspace, st);
    if (act == FF_RELU) return narrow_run<T, KD, true, true>(x, wg, wu, wd, dy, M, D, F, act, out, workspace, st);
    return narrow_run<T, KD, true, false>(x, wg, wu, wd, dy, M, D, F, act, out, workspace, st);
}
template <typename T>
int narrow_kd(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, int64_t M, int D, int F, int act, void* out, void* workspace, hipStream_t st) {
    return D <= 32 ? narrow_way<T, 1>(x, wg, wu, wd, dy, M, D, F, act, out, workspace, st) : narrow_way<T, 2>(x, wg, wu, wd, dy, M, D, F, act, out, workspace, st);
}

}  // namespace

// A workgroup walks all features for its 128 rows: where those are many and the rows few, the products of nf_gated_ff.hip, which split the features over the chip, are faster.
// A chunk takes 2 to 4 us, so 16 of them what the products' launches take at their smallest; from 16384 rows on half the CUs are busy here.
bool ff_narrow_fits(int64_t rows, int dim, int hidden) { return dim <= 64 && (hidden <= 512 || rows >= 16384); }

int64_t ff_narrow_workspace_bytes(int dim, int hidden, int dtype, bool backward) {
    return (int64_t)((hidden + 31) / 32) * (narrow_records(dim <= 32 ? 1 : 2, backward) * (dtype == FF_F32 ? 3 : 1) * 1024 + (backward ? 128 : 0));
}

// dy null: out = the block of x; else out = dx
int ff_narrow(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, int64_t rows, int dim, int hidden, int dtype, int act, void* out, void* workspace,
              hipStream_t st) {
    const auto f = dtype == FF_F32 ? narrow_kd<float> : dtype == FF_BF16 ? narrow_kd<ff_bf16> : narrow_kd<ff_half>;
    return f(x, wg, wu, wd, dy, rows, dim, hidden, act, out, workspace, st);
}
