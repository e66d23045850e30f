// The gated feed-forward block on 8-bit operands (e4m3 with a power-of-two scale per 32 values along k: nf_ff.h), forward only:
// h = act(x Wg^T) * (x Wu^T) is brought to the same form in the output stage of its product -- there 8 neighbouring lanes hold the 32 features of a block of a row, so that its
// maximum is three exchanges -- and out = h Wd^T is made from it.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies the scales in: lane l holds row l mod 32, k = 16 (l / 32) .. + 15 and 32 + 16 (l / 32) .. + 15 of the
// instruction's 64, and its scale operand is that of the row's block l / 32 (k 0 .. 31 or 32 .. 63).  A k step of the tile is 128 values: 128
// bytes of a row, as in the 16-bit kernels, whose loader moves them (two values as one 16-bit element), and 4 scale bytes of a row, one word.
//
// That instruction aligns the products of 16 consecutive k to the largest of them and drops what lies below 2^-12 of it (probed: beside a product
// of 2^16 one of 2^4 counts, one of 2^2 does not): about 1e-4 of a sum of products like a network's, which moves a few of h's values to a
// neighbouring step.  Beside a bfloat16 result's rounding that is small (0.0020 against 0.0017 from the exact sums at 4096 x 4096 x 8192); beside a float16
// or float32 result's it is not.  For those the values are multiplied as bfloat16, which holds value and scale exactly, on
// v_mfma_f32_32x32x16_bf16: float32 sums, at half the rate; v_cvt_scalef32_pk_bf16_fp8 makes two operands of two values and their scale.
//
// 4096 x 4096 x 8192: gate and up 305 us (1.8 PFLOP/s), down 131 us (2.1; a library product of 8192^3 2.65): two waves a SIMD whose fragment reads wait in front of their
// products -- put between them, as the 16-bit kernels do, they need more registers than there are (as it is, 2 and 5 of a lane's offsets wait in scratch memory and one or two come
// back every step).  4 x 4096 x 8192: 22 and 11 us, 3 TB/s of weights.
#include "nf_ff_gemm.h"
#include "nf_ff_rows.h"

typedef int ff_i32x8 __attribute__((ext_vector_type(8)));

static __device__ unsigned ff_unit_scales = 0x7f7f7f7fu;          // four scales of 1

namespace {

struct FfScales {
    const uint8_t *a, *b;          // gated: gate and up
    int64_t pitch;                 // bytes: k / 32
    int rows;
};

// the 4 scale bytes of blocks blk .. blk + 3 of a row; blocks behind the last have the scale 1 (their values are zeros)
__device__ __forceinline__ unsigned ff_scale_word(const uint8_t* row, int blk, int blocks) {
    if (blk + 4 <= blocks) {
        typedef unsigned U __attribute__((aligned(1)));
        return *reinterpret_cast<const U*>(row + blk);
    }
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (blk + i < blocks ? (unsigned)row[blk + i] : 127u) << (8 * i);
    return w;
}

// A step is 128 values of k (128-byte rows) in two halves of one instruction's 64, two stages, as in k_ff_gemm; a row's four scales of a step are one word, which comes by a 4-byte
// LDS-DMA a row, into a ring of its own (rows of words need a pitch of 4 bytes: the host pads other lengths with scales of 1).
// EXACT: the products in bfloat16
template <int BP, int BQ, int WP, int WQ, bool GATED, bool EXACT, typename Epi>
__global__ void __launch_bounds__(WP* WQ * 64) k_ff_gemm8(FfOperand p, FfOperand q, FfScales sp, FfScales sq, FfShape s, Epi epi) {
    constexpr int BK = 64;          // in pairs of values
    constexpr int WAVES = WP * WQ, SP = BP / WP, SQ = BQ / WQ, TP = SP / 32, TQ = SQ / 32;
    typedef FfLoader<1, BP, BK, WAVES, false, GATED, SP> LP;
    typedef FfLoader<1, BQ, BK, WAVES, false, false, SQ> LQ;
    constexpr int BUF = LP::BYTES + LQ::BYTES, LOADS = LP::PER_WAVE + LQ::PER_WAVE, SCALES = 2 * BUF, WORDS = (BP + BQ) * 4;
    static_assert(BP + BQ == WAVES * 64, "a wave moves the words of 64 rows");
    HIP_DYNAMIC_SHARED(char, lds)
    const int lane = threadIdx.x & 63, wave = ff_wave_index(), r32 = lane & 31, half = lane >> 5;
    const int wp = wave % WP, wq = wave / WP;
    int tm, tn;
    ff_tile_of(s, blockIdx.x, tm, tn);
    const int m0 = tm * BQ, n0 = tn * (GATED ? BP / 2 : BP);
    const int K = s.K;          // pairs of values
    const int words = (K + 63) / 64;
    LP lp;
    LQ lq;
    lp.init(p, n0, wave, lane);
    lq.init(q, m0, wave, lane);
    const uint8_t* srow;          // the row whose words this lane moves
    {
        const int v = wave * 64 + lane;
        if (v < BP) {
            const int in = v % SP;
            int row = GATED ? n0 + (v / SP) * (SP / 2) + in % (SP / 2) : n0 + v;
            if (row >= sp.rows) row = sp.rows - 1;
            srow = (GATED && in >= SP / 2 ? sp.b : sp.a) + row * sp.pitch;
        } else {
            int row = m0 + v - BP;
            if (row >= sq.rows) row = sq.rows - 1;
            srow = sq.a + row * sq.pitch;
        }
    }
    auto load_scales = [&](int word) {          // (a word behind the end is not used: its values are zeros, and the scales must be no NaN)
        const void* src = word < words ? (const void*)(srow + 4 * word) : (const void*)&ff_unit_scales;
        ff_dma4(src, lds, SCALES + (word & 1) * WORDS + wave * 256, lane);
    };
    ff_f32x16 acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        load_scales(t);
        lp.load(lds, t * BUF, t * BK, K, wave, lane);
        lq.load(lds, t * BUF + LP::BYTES, t * BK, K, wave, lane);
    }
    // one set of fragments: each is read again, for the next half, behind its last product
    ff_u32x4 a[TP][2], b[TQ][2];
    unsigned pw[TP], qw[TQ];
    auto fragment = [&](int row32, int at, int h, int c) {          // part c of half h of a row: k 64 h + 32 c + 16 (lane / 32) .. + 15
        const int r = row32 + r32;
        return *reinterpret_cast<const ff_u32x4*>(lds + at + r * (BK * 2) + (((4 * h + 2 * c + half) ^ ff_swz_inner<8>(r)) << 4));
    };
    auto read_p = [&](int i, int at, int h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) a[i][c] = fragment(wp * SP + 32 * i, at, h, c);
    };
    auto read_q = [&](int j, int at, int h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) b[j][c] = fragment(wq * SQ + 32 * j, at + LP::BYTES, h, c);
    };
    auto word = [&](int row, int slot) {
        const unsigned w = *reinterpret_cast<const unsigned*>(lds + SCALES + slot * WORDS + 4 * row);
        return EXACT ? w : w >> (8 * half);          // the instruction takes byte 0 (first half) or 2 (second) of the lane's word: its own block's
    };
    auto multiply = [&](auto which, int i, int j) {
        constexpr int h = decltype(which)::value;
        if constexpr (EXACT) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ff_from_e4m3x8(a[i][c][2 * e], a[i][c][2 * e + 1], (pw[i] >> (8 * (2 * h + c))) & 255u),
                                                                        ff_from_e4m3x8(b[j][c][2 * e], b[j][c][2 * e + 1], (qw[j] >> (8 * (2 * h + c))) & 255u),
                                                                        acc[i][j], 0, 0, 0);
        } else {
            const ff_i32x8 av = __builtin_bit_cast(ff_i32x8, a[i]), bv = __builtin_bit_cast(ff_i32x8, b[j]);
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[i][j], 0, 0, 2 * h, (int)pw[i], 2 * h, (int)qw[j]);
        }
    };
    ff_dma_barrier<LOADS + 1>();
#pragma unroll
    for (int j = 0; j < TQ; ++j) read_q(j, 0, 0);
#pragma unroll
    for (int i = 0; i < TP; ++i) read_p(i, 0, 0);
    int cur = 0;
    auto products = [&](auto which, auto whole, int read_at, int load_k) {
        constexpr int h = decltype(which)::value, PRODUCTS = TP * TQ;
#pragma unroll
        for (int j = 0; j < TQ; ++j)
#pragma unroll
            for (int i = 0; i < TP; ++i) {
                const int m = j * TP + i;
                multiply(which, i, j);
                if (h == 1) {
#pragma unroll
                    for (int n = m * LOADS / PRODUCTS; n < (m + 1) * LOADS / PRODUCTS; ++n) {
                        if (n < LP::PER_WAVE) lp.template issue<decltype(whole)::value>(n, lds, cur * BUF, load_k, K, wave, lane);
                        else lq.template issue<decltype(whole)::value>(n - LP::PER_WAVE, lds, cur * BUF + LP::BYTES, load_k, K, wave, lane);
                    }
                }
                if (j == TQ - 1) read_p(i, read_at, h ^ 1);
                if (i == TP - 1) {
                    read_q(j, read_at, h ^ 1);
                    if (!EXACT) ff_keep_order();          // (behind each product the fixed order costs registers that are not there)
                }
            }
    };
    auto step = [&](auto whole, int k0) {
#pragma unroll
        for (int i = 0; i < TP; ++i) pw[i] = word(wp * SP + 32 * i + r32, cur);
#pragma unroll
        for (int j = 0; j < TQ; ++j) qw[j] = word(BP + wq * SQ + 32 * j + r32, cur);
        products(std::integral_constant<int, 0>(), whole, cur * BUF, 0);
        ff_dma_barrier<0>();          // the tile has been read, the next one has landed
        load_scales(k0 / BK + 2);
        products(std::integral_constant<int, 1>(), whole, (cur ^ 1) * BUF, k0 + 2 * BK);
        cur ^= 1;
    };
    int k0 = 0;
    for (; k0 + 3 * BK <= K; k0 += BK) step(std::true_type(), k0);
    for (; k0 < K; k0 += BK) step(std::false_type(), k0);
    ff_dma_barrier<0>();          // no load may land in LDS that the workgroup has given back
    ff_output<BP, BQ, WP, WQ, GATED>(reinterpret_cast<float*>(lds), acc, s, m0, n0, 0, epi);
}

// rows of scales -> rows of `pitch` bytes (a multiple of 4), scales of 1 behind the end
__global__ void __launch_bounds__(256) k_ff_pad_scales(const uint8_t* __restrict__ src, int64_t rows, int blocks, int pitch, uint8_t* __restrict__ dst) {
    const int64_t n = rows * pitch;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / pitch;
        const int c = (int)(i - r * pitch);
        dst[i] = c < blocks ? src[r * blocks + c] : (uint8_t)127;
    }
}

// few rows (nf_ff_rows.h): 128 values of k a unit, whose scales are a word a row; 16 values a lane and step, as two bfloat16 operands.  The gated form has 32 weight rows
// a workgroup, so that the features of an h block are one workgroup's
constexpr int ff_rows8_most(int nt, bool gated) { return gated && nt >= 3 ? 4 : 8; }          // 64 KB of LDS at most
template <int NT, bool GATED, typename T>
__global__ void __launch_bounds__(64 * ff_rows8_most(NT, GATED)) k_ff_rows8(const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1, FfScales sw, const uint8_t* __restrict__ x,
                                                   const uint8_t* __restrict__ xs, int M, int N, int K, T* __restrict__ out, uint8_t* __restrict__ hq,
                                                   uint8_t* __restrict__ hs, int act) {
    constexpr int NW = GATED ? 2 : 1, HG = GATED ? 2 : 1, U = 2, UNIT = 128;
    HIP_DYNAMIC_SHARED(ff_f32x4, part)
    const int t0 = blockIdx.y * 16 * NT;          // this workgroup's first token
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16 * HG, blocks = K / 32;
    const uint8_t *wr[NW][HG], *ws[NW][HG], *xr[NT], *xsr[NT];
#pragma unroll
    for (int h = 0; h < HG; ++h) {          // (N is a multiple of 32)
        const int64_t n = n0 + 16 * h + r;
        wr[0][h] = w0 + n * K;
        ws[0][h] = sw.a + n * sw.pitch;
        if (GATED) {
            wr[NW - 1][h] = w1 + n * K;
            ws[NW - 1][h] = sw.b + n * sw.pitch;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t m = t0 + 16 * t + r < M ? t0 + 16 * t + r : M - 1;
        xr[t] = x + m * K;
        xsr[t] = xs + m * blocks;
    }
    ff_f32x4 acc[NW][HG][NT];
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][h][t] = ff_f32x4{0.f, 0.f, 0.f, 0.f};
    ff_u32x4 a[2][U][NW][HG], b[2][U][NT];
    unsigned as[2][NW][HG], bs[2][NT];
    auto fetch = [&](int s, int k0) {
        const ff_u32x4 none = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int k = k0 + 64 * j + 16 * q;
            const bool in = k < K;
#pragma unroll
            for (int i = 0; i < NW; ++i)
#pragma unroll
                for (int h = 0; h < HG; ++h) a[s][j][i][h] = in ? *reinterpret_cast<const ff_u32x4*>(wr[i][h] + k) : none;
#pragma unroll
            for (int t = 0; t < NT; ++t) b[s][j][t] = in ? *reinterpret_cast<const ff_u32x4*>(xr[t] + k) : none;
        }
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int h = 0; h < HG; ++h) as[s][i][h] = ff_scale_word(ws[i][h], k0 / 32, blocks);
#pragma unroll
        for (int t = 0; t < NT; ++t) bs[s][t] = ff_scale_word(xsr[t], k0 / 32, blocks);
    };
    auto multiply = [&](int s) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int sh = 8 * (2 * j + (q >> 1));
#pragma unroll
            for (int p = 0; p < 2; ++p) {          // bytes 0 .. 7 and 8 .. 15 of the lane's 16
                ff_bf16x8 bv[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) bv[t] = ff_from_e4m3x8(b[s][j][t][2 * p], b[s][j][t][2 * p + 1], (bs[s][t] >> sh) & 255u);
#pragma unroll
                for (int i = 0; i < NW; ++i)
#pragma unroll
                    for (int h = 0; h < HG; ++h) {
                        const ff_bf16x8 av = ff_from_e4m3x8(a[s][j][i][h][2 * p], a[s][j][i][h][2 * p + 1], (as[s][i][h] >> sh) & 255u);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[i][h][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv[t], acc[i][h][t], 0, 0, 0);
                    }
            }
        }
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
    constexpr int FRAGS = NW * HG * NT;
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int h = 0; h < HG; ++h)
#pragma unroll
            for (int t = 0; t < NT; ++t) part[(wave * FRAGS + (i * HG + h) * NT + t) * 64 + lane] = acc[i][h][t];
    __syncthreads();
    for (int t = wave; t < NT; t += waves) {
        const int m = t0 + 16 * t + r;
        ff_f32x4 v[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) v[h] = ff_rows_total(part, waves, FRAGS, h * NT + t, lane);
        if (GATED) {
            float top = 0.f;
            bool bad = false;
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                const ff_f32x4 u = ff_rows_total(part, waves, FRAGS, ((NW - 1) * HG + h) * NT + t, lane);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float ac, slope;
                    ff_act(act, v[h][c], ac, slope);
                    v[h][c] = ac * u[c];
                    top = fmaxf(top, fabsf(v[h][c]));
                    bad |= !(fabsf(v[h][c]) <= 3.4028235e38f);
                }
            }
            if (bad) top = INFINITY;
            top = fmaxf(top, __shfl_xor(top, 16, NF_WAVE));          // the 32 features of a token are on 4 lanes
            top = fmaxf(top, __shfl_xor(top, 32, NF_WAVE));
            const unsigned byte = ff_scale_byte(top);
            const float inv = byte == 255u ? NAN : ff_scale_inverse(byte);
            if (m < M) {
#pragma unroll
                for (int h = 0; h < HG; ++h)
                    *reinterpret_cast<unsigned*>(hq + (int64_t)m * N + n0 + 16 * h + 4 * q) =
                        ff_e4m3x4(v[h][0] * inv, v[h][1] * inv, v[h][2] * inv, v[h][3] * inv);
                if (q == 0) hs[(int64_t)m * (N / 32) + blockIdx.x] = (uint8_t)byte;
            }
        } else if (m < M) {
            typedef T V4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int h = 0; h < HG; ++h)
                *reinterpret_cast<V4*>(out + (int64_t)m * N + n0 + 16 * h + 4 * q) = V4{(T)v[h][0], (T)v[h][1], (T)v[h][2], (T)v[h][3]};
        }
    }
}

template <int NT, bool GATED, typename T>
void rows8(const void* w0, const void* w1, const FfScales& sw, const void* x, const uint8_t* xs, int M, int N, int K, T* out, uint8_t* hq, uint8_t* hs, int act,
           hipStream_t st) {
    constexpr int ROWS = GATED ? 32 : 16;
    const int waves = ff_rows_waves(N / ROWS, (K + 127) / 128, ff_rows8_most(NT, GATED));
    hipLaunchKernelGGL((k_ff_rows8<NT, GATED, T>), dim3(N / ROWS, (M + 16 * NT - 1) / (16 * NT)), dim3(64 * waves), (size_t)waves * (GATED ? 4 : 1) * NT * 1024, st,
                       (const uint8_t*)w0, (const uint8_t*)w1, sw, (const uint8_t*)x, xs, M, N, K, out, hq, hs, act);
}
template <bool GATED, typename T>
void few_rows8(const void* w0, const void* w1, const FfScales& sw, const void* x, const uint8_t* xs, int M, int N, int K, T* out, uint8_t* hq, uint8_t* hs, int act,
               hipStream_t st) {
    switch (ff_rows_tokens(M, N / (GATED ? 32 : 16))) {
        case 1: rows8<1, GATED, T>(w0, w1, sw, x, xs, M, N, K, out, hq, hs, act, st); break;
        case 2: rows8<2, GATED, T>(w0, w1, sw, x, xs, M, N, K, out, hq, hs, act, st); break;
        case 3: rows8<3, GATED, T>(w0, w1, sw, x, xs, M, N, K, out, hq, hs, act, st); break;
        default: rows8<4, GATED, T>(w0, w1, sw, x, xs, M, N, K, out, hq, hs, act, st);
    }
}

template <typename T>
struct Epi8Store {
    T* out;
    int64_t pitch;
    __device__ __forceinline__ void plain(int, int m, int n, int, bool inside, const ff_f32x4& v) const {          // N is a multiple of 32
        typedef T V4 __attribute__((ext_vector_type(4)));
        if (inside) *reinterpret_cast<V4*>(out + m * pitch + n) = V4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    }
    __device__ __forceinline__ void gated(int, int, int, int, bool, const ff_f32x4&, const ff_f32x4&) const {}
};

struct Epi8Gate {
    uint8_t *q, *scale;
    int64_t F, scale_pitch;
    int act;
    // 8 neighbouring lanes hold the 32 features of a block
    __device__ __forceinline__ void gated(int, int m, int n, int, bool inside, const ff_f32x4& g, const ff_f32x4& u) const {
        float v[4], top = 0.f;
        bool bad = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float a, slope;
            ff_act(act, g[c], a, slope);
            v[c] = a * u[c];
            top = fmaxf(top, fabsf(v[c]));
            bad |= !(fabsf(v[c]) <= 3.4028235e38f);
        }
        if (bad) top = INFINITY;          // (fmaxf drops a NaN)
        top = nf_grp_reduce<8>(top, NfMax());
        if (!inside) return;
        const unsigned byte = ff_scale_byte(top);
        const float inv = byte == 255u ? NAN : ff_scale_inverse(byte);
        *reinterpret_cast<unsigned*>(q + m * F + n) = ff_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        if (n % 32 == 0) scale[m * scale_pitch + n / 32] = (uint8_t)byte;
        if (n + 4 == F)
            for (int64_t c = F / 32; c < scale_pitch; ++c) scale[m * scale_pitch + c] = 127;
    }
    __device__ __forceinline__ void plain(int, int, int, int, bool, const ff_f32x4&) const {}
};

template <int BP, int BQ, int WP, int WQ, bool GATED, bool EXACT, typename Epi>
int launch8(const FfOperand& p, const FfOperand& q, const FfScales& sp, const FfScales& sq, int M, int N, int K, const Epi& epi, hipStream_t st) {
    constexpr int RING = 2 * (BP + BQ) * 128 + 2 * (BP + BQ) * 4, OUT = ff_output_bytes<BP, BQ, WP, WQ>(), LDS = RING > OUT ? RING : OUT, COLS = GATED ? BP / 2 : BP;
    static bool set[NF_MAX_DEVICES];
    const int dev = nf_current_device();
    const auto kernel = k_ff_gemm8<BP, BQ, WP, WQ, GATED, EXACT, Epi>;
    if (!set[dev]) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            nf_set_error("gated feed-forward in 8 bits: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
            return 2;
        }
        set[dev] = true;
    }
    FfShape s;
    s.M = M, s.N = N, s.K = K / 2, s.n_end = N;
    s.tiles_m = (M + BQ - 1) / BQ, s.tiles_n = (N + COLS - 1) / COLS;
    s.k_part = K / 2;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(s.tiles_m * s.tiles_n)), dim3(WP * WQ * 64), LDS, st, p, q, sp, sq, s, epi);
    return 0;
}

// tile: 256 x 256 where that gives most of the 256 CUs a tile, else 128 x 128.  Rows x 4096 x 4096, gate and up on so many tiles of 256 (down half of them), us with 128 and 256: 128
// tiles 80 and 106, 160 tiles 108 and 106, 256 tiles 138 and 120, 512 tiles 261 and 201; with bfloat16 operands 113 and 161, 155 and 162, 199 and 190, 383 and 330.
bool big_tiles8(int64_t M, int64_t N) { return ((M + 255) / 256) * ((N + 255) / 256) >= 160; }
template <bool GATED, bool EXACT, typename Epi>
int product8(const FfOperand& p, const FfOperand& q, const FfScales& sp, const FfScales& sq, int M, int N, int K, const Epi& epi, hipStream_t st) {
    if (big_tiles8(M, N * (GATED ? 2 : 1))) return launch8<256, 256, 2, 4, GATED, EXACT>(p, q, sp, sq, M, N, K, epi, st);
    return launch8<128, 128, 2, 2, GATED, EXACT>(p, q, sp, sq, M, N, K, epi, st);
}

FfOperand operand8(const void* a, const void* b, int rows, int K) {
    return FfOperand{(const uint16_t*)a, (const uint16_t*)b, K / 2, rows, 0x7fffffff, 0x7fffffff};
}

// the workspace of the tiled form: h in 8 bits, and the scales whose rows are no multiple of 4 bytes
struct Plan8 {
    uint8_t *hq, *hs, *xs = nullptr, *gs = nullptr, *us = nullptr, *ds = nullptr;
    int64_t dp, fp;          // pitches of the scales of rows of D and F values
    int64_t bytes = 0;
    Plan8(uint8_t* base, int64_t M, int64_t D, int64_t F) {
        dp = (D / 32 + 3) / 4 * 4;
        fp = (F / 32 + 3) / 4 * 4;
        auto take = [&](int64_t n) {
            uint8_t* p = base ? base + bytes : nullptr;
            bytes += (n + 255) / 256 * 256;
            return p;
        };
        hq = take(M * F);
        hs = take(M * fp);
        if (dp != D / 32) xs = take(M * dp), gs = take(F * dp), us = take(F * dp);
        if (fp != F / 32) ds = take(D * fp);
    }
};
const uint8_t* padded_scales(const uint8_t* src, int64_t rows, int blocks, int64_t pitch, uint8_t* to, hipStream_t st) {
    if (pitch == blocks) return src;
    int64_t grid = (rows * pitch + 255) / 256;
    if (grid > 4096) grid = 4096;
    hipLaunchKernelGGL(k_ff_pad_scales, dim3((unsigned)grid), dim3(256), 0, st, src, rows, blocks, (int)pitch, to);
    return to;
}

bool sizes_ok8(const char* what, int64_t rows, int dim, int hidden, int out_dtype, int activation) {
    if (rows >= 1 && rows <= (1 << 30) && dim >= 32 && hidden >= 32 && dim % 32 == 0 && hidden % 32 == 0 && dim <= (1 << 20) && hidden <= (1 << 20) && out_dtype >= FF_F32 &&
        out_dtype <= FF_F16 && activation >= FF_SILU && activation <= FF_RELU)
        return true;
    nf_set_error("%s: need 1 <= rows <= 2^30, dim and hidden multiples of 32 up to 2^20, dtype and activation in 0 .. 2 (got rows %lld dim %d hidden %d dtype %d activation %d)", what,
                 (long long)rows, dim, hidden, out_dtype, activation);
    return false;
}

}  // namespace

extern "C" int64_t nf_gated_ff_fwd_8bit_workspace_bytes(int64_t rows, int dim, int hidden) {
    if (!sizes_ok8("nf_gated_ff_fwd_8bit_workspace_bytes", rows, dim, hidden, 0, 0)) return -1;
    return Plan8(nullptr, rows, dim, hidden).bytes;
}

extern "C" int nf_gated_ff_fwd_8bit(const void* x, const uint8_t* x_scale, const void* w_gate, const uint8_t* gate_scale, const void* w_up,
                                    const uint8_t* up_scale, const void* w_down, const uint8_t* down_scale, int64_t rows, int dim, int hidden,
                                    int out_dtype, int activation, void* out, void* workspace, nf_stream_t stream) {
    if (!sizes_ok8("nf_gated_ff_fwd_8bit", rows, dim, hidden, out_dtype, activation)) return 1;
    hipStream_t st = (hipStream_t)stream;
    const int M = (int)rows, D = dim, F = hidden;
    const Plan8 f((uint8_t*)workspace, rows, dim, hidden);
    // few rows: as FF_ROWS_MAX (nf_gated_ff.hip); 4096 x 8192, us: 16 rows 36 (tiles 70), 64 rows 61 (73), 65 rows 95 (73), 128 rows 116 (78)
    if (M <= 64) {
        const FfScales spg = {gate_scale, up_scale, D / 32, F};
        few_rows8<true, float>(w_gate, w_up, spg, x, x_scale, M, F, D, nullptr, f.hq, f.hs, activation, st);
        const FfScales sd = {down_scale, down_scale, F / 32, D};
        if (out_dtype == FF_F32) few_rows8<false, float>(w_down, nullptr, sd, f.hq, f.hs, M, D, F, (float*)out, nullptr, nullptr, 0, st);
        else if (out_dtype == FF_BF16) few_rows8<false, ff_bf16>(w_down, nullptr, sd, f.hq, f.hs, M, D, F, (ff_bf16*)out, nullptr, nullptr, 0, st);
        else few_rows8<false, ff_half>(w_down, nullptr, sd, f.hq, f.hs, M, D, F, (ff_half*)out, nullptr, nullptr, 0, st);
        NF_LAUNCH_CHECK("nf_gated_ff_fwd_8bit");
        return 0;
    }
    const FfOperand pg = operand8(w_gate, w_up, F, D), qx = operand8(x, x, M, D);
    const FfScales sqx = {padded_scales(x_scale, M, D / 32, f.dp, f.xs, st), nullptr, f.dp, M};
    const FfScales spg = {padded_scales(gate_scale, F, D / 32, f.dp, f.gs, st), padded_scales(up_scale, F, D / 32, f.dp, f.us, st), f.dp, F};
    int rc = out_dtype == FF_BF16 ? product8<true, false>(pg, qx, spg, sqx, M, F, D, Epi8Gate{f.hq, f.hs, F, f.fp, activation}, st)
                                  : product8<true, true>(pg, qx, spg, sqx, M, F, D, Epi8Gate{f.hq, f.hs, F, f.fp, activation}, st);
    if (rc) return rc;
    const FfOperand p = operand8(w_down, w_down, D, F), q = operand8(f.hq, f.hq, M, F);
    const FfScales sp = {padded_scales(down_scale, D, F / 32, f.fp, f.ds, st), nullptr, f.fp, D}, sq = {f.hs, f.hs, f.fp, M};
    if (out_dtype == FF_F32) rc = product8<false, true>(p, q, sp, sq, M, D, F, Epi8Store<float>{(float*)out, D}, st);
    else if (out_dtype == FF_BF16) rc = product8<false, false>(p, q, sp, sq, M, D, F, Epi8Store<ff_bf16>{(ff_bf16*)out, D}, st);
    else rc = product8<false, true>(p, q, sp, sq, M, D, F, Epi8Store<ff_half>{(ff_half*)out, D}, st);
    if (rc) return rc;
    NF_LAUNCH_CHECK("nf_gated_ff_fwd_8bit");
    return 0;
}

extern "C" int nf_gated_ff_8bit_form(int64_t rows, int dim, int hidden, int product) {
    if (!sizes_ok8("nf_gated_ff_8bit_form", rows, dim, hidden, 0, 0)) return -1;
    if (product < 0 || product > 1) {
        nf_set_error("nf_gated_ff_8bit_form: product 0 or 1 (got %d)", product);
        return -1;
    }
    if (rows <= 64) return 0;
    return 1 << 16 | (big_tiles8(rows, product ? dim : 2 * (int64_t)hidden) ? 256 : 128);
}
