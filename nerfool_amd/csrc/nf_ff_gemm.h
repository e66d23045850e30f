// The tiled matrix product of the gated feed-forward block: C[m][n] = sum over k of Q[m][k] P[n][k] on the bf16 / f16 matrix cores, with the
// element-wise work of the block in its output stage.
//
// Operands (16-bit, NP planes: 1, or 3 for a float32 operand held as three bf16 parts, whose six products of order <= 2^-16 give float32-grade sums):
//   k innermost    row r at a + r * pitch, k contiguous.  A gated P has two sources: the features' gate rows in a and their up rows in b.
//   k outermost    row k at a + k * pitch (k < seg) or b + (k - seg) * pitch, the product's n or m contiguous: the gradients' products read the
//                  tensors as they lie, the transposition happens in the LDS read (ds_read_b64_tr_b16).
// Tiles go global -> LDS by LDS-DMA, 16 bytes a lane, one k step ahead of their use; nothing passes through registers.  A lane whose 16 bytes lie
// behind the end of k, n or m reads a page of zeros instead (k, and n or m where they are contiguous, are multiples of 8: the host pads what is not).
// The 16-byte chunks of a row are placed at (chunk ^ f(row)), so that neither the plain nor the transposed reads collide in the LDS banks; the
// DMA writes lanes in order, hence the permutation is applied to the address that a lane reads.
//
// P is the A operand of v_mfma_f32_32x32x16 (rows in registers), Q the B operand (columns on lanes): a lane ends with one m and 4 consecutive n.
#pragma once

#include "nf_ff.h"

struct FfOperand {
    const uint16_t *a, *b;
    int64_t plane, pitch;          // elements
    int rows;                      // n or m
    int len, seg;                  // k outermost: rows k < len are a's, rows k >= seg are b's, rows between are zeros
};

static __device__ ff_u32x4 ff_zero_page = {0u, 0u, 0u, 0u};

// one LDS-DMA: the wave's lane l moves 16 bytes from its own address to dst + 16 l
__device__ __forceinline__ void ff_dma16(const void* src, char* dst, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    unsigned keep;
    const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
                 : "memory");
#else
    __builtin_memcpy(dst + 16 * lane, src, 16);
#endif
}
// all of this wave's LDS-DMAs have landed
__device__ __forceinline__ void ff_dma_wait() {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#endif
}

// 16 lanes read a 4 (k) x 16 block whose rows are k; lane i gets its column i as 4 consecutive k.  Lane i's address: k = i / 4, columns 4 (i % 4) ..
__device__ __forceinline__ uint64_t ff_read_tr(const char* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p)));
#elif defined(NF_HIP_EMU)
    return nf_emu_read_tr16(p);
#else
    (void)p;
    return 0;
#endif
}

template <typename E>
struct FfMfma;
template <>
struct FfMfma<ff_bf16> {
    typedef ff_bf16x8 V;
    static __device__ __forceinline__ ff_f32x16 mul(V a, V b, ff_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct FfMfma<ff_half> {
    typedef ff_half8 V;
    static __device__ __forceinline__ ff_f32x16 mul(V a, V b, ff_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// where chunk c (16 bytes) of row r of an LDS tile lies; CH chunks a row
template <int CH>
__device__ __forceinline__ int ff_swz_inner(int r) {          // rows are n or m, read 32 rows x one chunk at a time
    return CH == 8 ? (r & 7) : ((r >> 2) & 3);
}
template <int CH>
__device__ __forceinline__ int ff_swz_outer(int k) {          // rows are k, read 4 rows x 32 bytes a quarter wave
    return CH >= 16 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
}

// one operand's share of the tile loads of a wave
template <int NP, int ROWS, int BK, int WAVES, bool OUTER, bool GATED, int WSPAN>
struct FfLoader {
    static constexpr int CH = OUTER ? ROWS / 8 : BK / 8;                     // chunks of an LDS row
    static constexpr int PIECES = ROWS * BK * 2 / 1024;                       // 1 KB pieces of a plane's tile
    static constexpr int PER_WAVE = NP * PIECES / WAVES;
    static constexpr int RPP = 64 / CH;                                       // LDS rows a piece
    static constexpr int BYTES = NP * PIECES * 1024;
    static_assert(NP * PIECES % WAVES == 0, "every wave moves the same number of pieces");
    const uint16_t* ptr[PER_WAVE];
    int64_t step, jump;
    int kc, len, seg;     // kc: this lane's k inside the tile (k innermost)
    unsigned valid;       // outer: whether the column exists

    __device__ __forceinline__ void init(const FfOperand& o, int row0, int k0, int wave, int lane) {
        const int slot = lane % CH, rr = lane / CH;
        len = o.len;
        seg = o.seg;
        jump = OUTER ? (o.b - o.a) - (int64_t)o.seg * o.pitch : 0;
        step = OUTER ? (int64_t)BK * o.pitch : BK;
        valid = 0;
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
            const int li = wave * PER_WAVE + i, plane = li / PIECES, r = (li % PIECES) * RPP + rr;
            if (OUTER) {
                const int col = row0 + 8 * (slot ^ ff_swz_outer<CH>(r));
                if (col < o.rows) valid |= 1u << i;
                ptr[i] = o.a + plane * o.plane + (int64_t)(k0 + r) * o.pitch + col;
            } else {
                const int chunk = slot ^ ff_swz_inner<CH>(r);
                kc = 8 * chunk;          // (r mod 8, r / 4 mod 4 do not depend on the piece)
                const uint16_t* base = o.a;
                int row;
                if (GATED) {          // a wave's WSPAN rows: half gate, half up, of the same features
                    const int in = r % WSPAN;
                    row = row0 + (r / WSPAN) * (WSPAN / 2) + in % (WSPAN / 2);
                    if (in >= WSPAN / 2) base = o.b;
                } else
                    row = row0 + r;
                if (row >= o.rows) row = o.rows - 1;          // a row behind the end: any values, its results are not stored
                ptr[i] = base + plane * o.plane + (int64_t)row * o.pitch + k0 + kc;
            }
        }
    }
    // the tile at k0 (which the pointers stand at) -> buf
    __device__ __forceinline__ void load(char* buf, int k0, int K, int wave, int lane) {
        const int rr = lane / CH;
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
            const int li = wave * PER_WAVE + i;
            const void* src;
            if (OUTER) {
                const int k = k0 + (li % PIECES) * RPP + rr;
                src = k < K && (k < len || k >= seg) && ((valid >> i) & 1u) ? (const void*)(ptr[i] + (k >= seg ? jump : 0)) : (const void*)&ff_zero_page;
            } else
                src = k0 + kc < K ? (const void*)ptr[i] : (const void*)&ff_zero_page;
            ff_dma16(src, buf + li * 1024, lane);
            ptr[i] += step;
        }
    }
};

// the 8 k of a fragment: row `row` (of this lane) of the tile plane at `tile`, k block kk of 16
template <typename V, int ROWS, int BK, bool OUTER>
__device__ __forceinline__ V ff_fragment(const char* tile, int row32, int kk, int lane) {
    constexpr int CH = OUTER ? ROWS / 8 : BK / 8;
    if (!OUTER) {
        const int r = row32 + (lane & 31), chunk = 2 * kk + (lane >> 5);
        return *reinterpret_cast<const V*>(tile + r * (BK * 2) + ((chunk ^ ff_swz_inner<CH>(r)) << 4));
    } else {
        // quarter wave g: rows 16 (g & 1) .., k 8 (g >> 1) ..; two transposed reads of 4 k
        const int i = lane & 15, col = row32 + ((lane >> 4) & 1) * 16 + (i & 3) * 4, k = 16 * kk + (lane >> 5) * 8 + (i >> 2);
        uint64_t t[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int kr = k + 4 * s;
            t[s] = ff_read_tr(tile + kr * (ROWS * 2) + (((col >> 3) ^ ff_swz_outer<CH>(kr)) << 4) + (col & 7) * 2);
        }
        V v;
        __builtin_memcpy(&v, t, 16);
        return v;
    }
}

struct FfShape {
    int M, N, K;           // N: columns of the result (features for the gated form)
    int n_end;             // columns N .. n_end - 1 are stored as zeros (the padding of an operand of a later product)
    int tiles_m, tiles_n;
    int k_split;           // k is cut into this many parts of k_part (a multiple of the k step)
    int k_part;
};

// Workgroup -> tile.  Consecutive workgroups go to the 8 XCDs in turn: each XCD gets a contiguous run of the tile order, so that its L2 keeps
// the operand strips that neighbouring tiles share; inside a run, groups of 8 tile rows (m) are walked column by column.
__device__ __forceinline__ void ff_tile_of(const FfShape& s, int id, int& tm, int& tn) {
    const int n = s.tiles_m * s.tiles_n, q = n / 8, r = n % 8, x = id % 8, y = id / 8;
    const int t = x * q + (x < r ? x : r) + y;
    const int span = 8 * s.tiles_n, g = t / span, in = t - g * span;
    const int rows = s.tiles_m - 8 * g < 8 ? s.tiles_m - 8 * g : 8;
    tm = 8 * g + in % rows;
    tn = in / rows;
}

// tile BP (rows of P) x BQ (rows of Q), WP x WQ waves
template <typename E, int NP, int BP, int BQ, int WP, int WQ, int BK, bool PO, bool QO, bool GATED, typename Epi>
__global__ void __launch_bounds__(WP* WQ * 64) k_ff_gemm(FfOperand p, FfOperand q, FfShape s, Epi epi) {
    typedef typename FfMfma<E>::V V;
    constexpr int WAVES = WP * WQ, SP = BP / WP, SQ = BQ / WQ, TP = SP / 32, TQ = SQ / 32;
    typedef FfLoader<NP, BP, BK, WAVES, PO, GATED, SP> LP;
    typedef FfLoader<NP, BQ, BK, WAVES, QO, false, SQ> LQ;
    constexpr int BUF = LP::BYTES + LQ::BYTES;
    HIP_DYNAMIC_SHARED(char, lds)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wp = wave % WP, wq = wave / WP;
    const int tiles = s.tiles_m * s.tiles_n, part = blockIdx.x / tiles;
    int tm, tn;
    ff_tile_of(s, blockIdx.x - part * tiles, tm, tn);
    const int m0 = tm * BQ, n0 = tn * (GATED ? BP / 2 : BP);
    const int k_lo = part * s.k_part, k_hi = k_lo + s.k_part < s.K ? k_lo + s.k_part : s.K;
    LP lp;
    LQ lq;
    lp.init(p, n0, k_lo, wave, lane);
    lq.init(q, m0, k_lo, wave, lane);
    ff_f32x16 acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    lp.load(lds, k_lo, k_hi, wave, lane);
    lq.load(lds + LP::BYTES, k_lo, k_hi, wave, lane);
    int cur = 0;
    for (int k0 = k_lo; k0 < k_hi; k0 += BK) {
        ff_dma_wait();
        __syncthreads();          // the tile has landed for every wave, and the other buffer has been read by every wave
        if (k0 + BK < k_hi) {
            char* nb = lds + (cur ^ 1) * BUF;
            lp.load(nb, k0 + BK, k_hi, wave, lane);
            lq.load(nb + LP::BYTES, k0 + BK, k_hi, wave, lane);
        }
        const char* bp = lds + cur * BUF;
        const char* bq = bp + LP::BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
            V a[NP][TP], b[NP][TQ];
#pragma unroll
            for (int e = 0; e < NP; ++e) {
#pragma unroll
                for (int i = 0; i < TP; ++i) a[e][i] = ff_fragment<V, BP, BK, PO>(bp + e * (LP::BYTES / NP), wp * SP + 32 * i, kk, lane);
#pragma unroll
                for (int j = 0; j < TQ; ++j) b[e][j] = ff_fragment<V, BQ, BK, QO>(bq + e * (LQ::BYTES / NP), wq * SQ + 32 * j, kk, lane);
            }
            // smallest products first
#pragma unroll
            for (int o = NP - 1; o >= 0; --o)
#pragma unroll
                for (int e = 0; e <= o; ++e)
#pragma unroll
                    for (int i = 0; i < TP; ++i)
#pragma unroll
                        for (int j = 0; j < TQ; ++j) acc[i][j] = FfMfma<E>::mul(a[e][i], b[o - e][j], acc[i][j]);
        }
        cur ^= 1;
    }
    // lane: m = the lane's column, n = 8 g + 4 (lane / 32) + 0 .. 3 of each 32 x 32 block
    const int h = lane >> 5;
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        const int m = m0 + wq * SQ + 32 * j + (lane & 31);
        if (m >= s.M) continue;
        if (GATED) {
#pragma unroll
            for (int i = 0; i < TP / 2; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = n0 + wp * (SP / 2) + 32 * i + 8 * g + 4 * h;
                    float v[4], u[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        v[c] = acc[i][j][4 * g + c];
                        u[c] = acc[(i + TP / 2) % TP][j][4 * g + c];
                    }
                    if (n < s.n_end) epi.gated(part, m, n, s.N - n, v, u);
                }
        } else {
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = n0 + wp * SP + 32 * i + 8 * g + 4 * h;
                    float v[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c] = acc[i][j][4 * g + c];
                    if (n < s.n_end) epi.plain(part, m, n, s.N - n, v);
                }
        }
    }
}
