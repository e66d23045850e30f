// The tiled matrix product of the gated feed-forward block: C[m][n] = sum over k of Q[m][k] P[n][k] on the bf16 / f16 matrix cores, with the
// element-wise work of the block in its output stage.
//
// Operands (16-bit, NP planes: 1, or 3 for a float32 operand held as three bf16 parts, whose six products of order <= 2^-16 give float32-grade sums):
// The three planes lie in blocks of 32 values along a row, [block][plane][32]: what a step of 32 k reads of a row is 192 bytes in one place (apart, the planes' 64 bytes were half
// cache lines each, and the L2 gave half its rate); rows are padded to a multiple of 32 values.
//   k innermost    row r at a + r * pitch, k contiguous.  A gated P has two sources: the features' gate rows in a and their up rows in b.
//   k outermost    row k at a + k * pitch (k < seg) or b + (k - seg) * pitch, the product's n or m contiguous: the gradients' products read the
//                  tensors as they lie, the transposition happens in the LDS read (ds_read_b64_tr_b16).
// Tiles go global -> LDS by LDS-DMA, 16 bytes a lane, one or two k steps ahead of their use; nothing passes through registers.  A lane whose 16 bytes lie
// behind the end of k reads a page of zeros instead, one behind the end of n or m the last rows or columns again (k, and n or m where they are contiguous, are
// multiples of 8: the host pads what is not).
// The 16-byte chunks of a row are placed at (chunk ^ f(row)), so that neither the plain nor the transposed reads collide in the LDS banks; the
// DMA writes lanes in order, hence the permutation is applied to the address that a lane reads.
//
// P is the A operand of v_mfma_f32_16x16x32 (rows in registers), Q the B operand (columns on lanes): a lane ends with one m and 4 consecutive n.
// The results go through LDS, 32 rows of every wave at a time, so that the output stage reads and writes whole rows: from the fragments directly a
// wave's 16-byte accesses lie in 16 or 32 rows, and the stage of dh's product (g, u in, three tensors out) took twice the time of its 64 k steps.
// The 256 x 256 form takes all 256 registers of its lanes; where an operand is k outermost (the backward pass) 2 to 6 of their load offsets wait in scratch memory and come back
// between the products of each step.
#pragma once

#include <type_traits>

#include "nf_ff.h"

struct FfOperand {
    const uint16_t *a, *b;
    int64_t pitch;                 // elements (of all planes)
    int rows;                      // n or m
    int len, seg;                  // k outermost: rows k < len are a's, rows k >= seg are b's, rows between are zeros
};

static __device__ ff_u32x4 ff_zero_page = {0u, 0u, 0u, 0u};

// one LDS-DMA: the wave's lane l moves 16 bytes from its own address to lds + at + 16 l (lds: the workgroup's dynamic LDS, at: the same for the wave)
__device__ __forceinline__ void ff_dma16(const void* src, char* lds, int at, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    unsigned keep;
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds + at);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(src), "s"(to)
                 : "memory");
#else
    __builtin_memcpy(lds + at + 16 * lane, src, 16);
#endif
}
// ... from base + off, off the lane's own, base the same for the wave
__device__ __forceinline__ void ff_dma16(const char* base, unsigned off, char* lds, int at, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    unsigned keep;
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds + at);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(to), "s"(base)
                 : "memory");
#else
    __builtin_memcpy(lds + at + 16 * lane, base + off, 16);
#endif
}
// ... 4 bytes a lane
__device__ __forceinline__ void ff_dma4(const void* src, char* lds, int at, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    unsigned keep;
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds + at);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(src), "s"(to)
                 : "memory");
#else
    __builtin_memcpy(lds + at + 4 * lane, src, 4);
#endif
}
// the compiler moves nothing across this
__device__ __forceinline__ void ff_keep_order() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
#endif
}
__device__ __forceinline__ int ff_wave_index() {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#else
    return threadIdx.x >> 6;
#endif
}
// at most N of this wave's LDS-DMAs are still under way (they land in order), its LDS reads have returned, and so it is for every wave of the workgroup
template <int N>
__device__ __forceinline__ void ff_dma_barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
#else
    __syncthreads();
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
    static __device__ __forceinline__ ff_f32x4 mul(V a, V b, ff_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct FfMfma<ff_half> {
    typedef ff_half8 V;
    static __device__ __forceinline__ ff_f32x4 mul(V a, V b, ff_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// where chunk c (16 bytes) of row r of an LDS tile lies; CH chunks a row
template <int CH>
__device__ __forceinline__ int ff_swz_inner(int r) {          // rows are n or m, read 32 rows x one chunk at a time
    return CH == 8 ? (r >> 1) & 7 : (r >> 2) & 3;          // (16 lanes of a read cover the 64 banks once)
}
template <int CH>
__device__ __forceinline__ int ff_swz_outer(int k) {          // rows are k, read 4 rows x 32 bytes a quarter wave, quarters 8 rows apart
    return (CH >= 16 ? (k & 3) << 2 : (k & 2) << 1) ^ (((k >> 3) & 1) << 1);
}

// One operand's share of the tile loads of a wave.  A lane keeps a 32-bit offset a load; what changes from tile to tile is the same for the wave.  A tile whose 16-byte
// pieces all exist (whole()) is loaded by these alone; another one, at the end of k or where a's rows end and b's begin, goes lane by lane, with zeros where nothing is.
template <int NP, int ROWS, int BK, int WAVES, bool OUTER, bool GATED, int WSPAN>
struct FfLoader {
    static constexpr int CH = OUTER ? ROWS / 8 : BK / 8;                     // chunks of an LDS row
    static constexpr int PIECES = ROWS * BK * 2 / 1024;                       // 1 KB pieces of a plane's tile
    static constexpr int PER_WAVE = NP * PIECES / WAVES;
    static constexpr int RPP = 64 / CH;                                       // LDS rows a piece
    static constexpr int BYTES = NP * PIECES * 1024;
    static_assert(NP * PIECES % WAVES == 0, "every wave moves the same number of pieces");
    static_assert(!GATED || (WSPAN / 2) % RPP == 0, "a piece's rows are of one source");
    static constexpr int PER_K = NP == 3 ? 6 : 2;                             // bytes a k
    unsigned off[PER_WAVE];
    const char *a, *b;
    int64_t pitch;          // bytes
    int len, seg;

    __device__ __forceinline__ void init(const FfOperand& o, int row0, int wave, int lane) {
        const int slot = lane % CH, rr = lane / CH;
        a = (const char*)o.a;
        b = (const char*)o.b;
        pitch = o.pitch * 2;
        len = o.len;
        seg = o.seg;
        if (!OUTER) {
            a += row0 * pitch;
            b += row0 * pitch;
        }
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
            const int li = wave * PER_WAVE + i, r = li % PIECES * RPP + rr, plane = li / PIECES;
            // a row, or columns, behind the end: the last ones, whose results are not stored
            if (OUTER) {
                int col = row0 + 8 * (slot ^ ff_swz_outer<CH>(r));
                if (col >= o.rows) col = o.rows - 8;
                off[i] = (unsigned)(r * pitch + (NP == 3 ? col / 32 * 192 + 64 * plane + col % 32 * 2 : 2 * col));
            } else {
                int row = GATED ? (r / WSPAN) * (WSPAN / 2) + r % (WSPAN / 2) : r;          // a wave's WSPAN rows: half gate, half up, of the same features
                if (row0 + row >= o.rows) row = o.rows - 1 - row0;
                off[i] = (unsigned)(row * pitch + 64 * plane + 16 * (slot ^ ff_swz_inner<CH>(r)));          // (one plane: plane 0)
            }
        }
    }
    __device__ __forceinline__ bool whole(int k0, int K) const { return k0 + BK <= K && (!OUTER || k0 >= seg || k0 + BK <= len); }
    // piece i of this wave of the tile at k0 -> lds + at
    template <bool WHOLE>
    __device__ __forceinline__ void issue(int i, char* lds, int at, int k0, int K, int wave, int lane) {
        const int li = wave * PER_WAVE + i;
        const char* base = GATED && li % PIECES * RPP % WSPAN >= WSPAN / 2 ? b : a;
        if (OUTER) base = k0 >= seg ? b + (k0 - seg) * pitch : a + k0 * pitch;
        else base += PER_K * (int64_t)k0;
        if (WHOLE) {
            ff_dma16(base, off[i], lds, at + li * 1024, lane);
        } else {
            const void* src = base + off[i];
            bool in;
            if (OUTER) {
                const int k = k0 + li % PIECES * RPP + lane / CH;
                in = k < K && (k < len || k >= seg);
                if (k0 < seg && k >= seg) src = (const char*)src + ((b - a) - seg * pitch);
            } else
                in = k0 + 8 * ((lane % CH) ^ ff_swz_inner<CH>(li % PIECES * RPP + lane / CH)) < K;
            ff_dma16(in ? src : (const void*)&ff_zero_page, lds, at + li * 1024, lane);
        }
    }
    __device__ __forceinline__ void load(char* lds, int at, int k0, int K, int wave, int lane) {
        if (whole(k0, K)) {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) issue<true>(i, lds, at, k0, K, wave, lane);
        } else {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) issue<false>(i, lds, at, k0, K, wave, lane);
        }
    }
};

// a 16 x 32 fragment of the tile plane at `tile`, k block kk of 32: lane l holds row row16 + l mod 16, k = 8 (l / 16) .. + 7
template <typename V, int ROWS, int BK, bool OUTER>
__device__ __forceinline__ V ff_fragment(const char* tile, int row16, int kk, int lane) {
    constexpr int CH = OUTER ? ROWS / 8 : BK / 8;
    if (!OUTER) {
        const int r = row16 + (lane & 15);
        return *reinterpret_cast<const V*>(tile + r * (BK * 2) + (((4 * kk + (lane >> 4)) ^ ff_swz_inner<CH>(r)) << 4));
    } else {
        // a quarter wave reads rows k = 8 (l / 16) + 4 s + i / 4, columns row16 + 4 (i % 4) .. + 3, and gets its transpose
        const int i = lane & 15, col = row16 + (i & 3) * 4, k = 32 * kk + (lane >> 4) * 8 + (i >> 2);
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
    int k_part;            // k is cut into parts of this length (a multiple of the k step)
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

// bytes of LDS that ff_output needs
template <int BP, int BQ, int WP, int WQ>
constexpr int ff_output_bytes() {
    return WQ * 32 * (BP + 4) * 4;
}
// The accumulators of a tile -> epi, 4 consecutive n of a row at a time: epi.plain(part, m, n, left, inside, v) or epi.gated(part, m, n, left, inside, gate, up), left = s.N - n.
// Every thread makes every call (epi may exchange values between neighbouring lanes, which hold neighbouring n of the row); inside: the place exists.
template <int BP, int BQ, int WP, int WQ, bool GATED, typename Acc, int TP, int TQ, typename Epi>
__device__ __forceinline__ void ff_output(float* lds, const Acc (&acc)[TP][TQ], const FfShape& s, int m0, int n0, int part, const Epi& epi) {
    constexpr bool SMALL = sizeof(Acc) == 16;          // 16 x 16 blocks, else 32 x 32
    constexpr int SP = BP / WP, SQ = BQ / WQ, PITCH = BP + 4, COLS = GATED ? BP / 2 : BP, THREADS = WP * WQ * 64, ITEMS = WQ * 32 * COLS / 4;
    static_assert(ITEMS % THREADS == 0, "every thread makes the same number of calls");
    const int lane = threadIdx.x & 63, wave = ff_wave_index(), wp = wave % WP, wq = wave / WP;
#pragma unroll
    for (int j = 0; j < SQ / 32; ++j) {
        if (j) __syncthreads();
        if constexpr (SMALL) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* row = lds + (wq * 32 + 16 * h + (lane & 15)) * PITCH + wp * SP + 4 * (lane >> 4);
#pragma unroll
                for (int i = 0; i < TP; ++i) *reinterpret_cast<ff_f32x4*>(row + 16 * i) = acc[i][2 * j + h];
            }
        } else {
            float* row = lds + (wq * 32 + (lane & 31)) * PITCH + wp * SP + 4 * (lane >> 5);
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<ff_f32x4*>(row + 32 * i + 8 * g) = ff_f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
        __syncthreads();
#pragma unroll 2
        for (int it = threadIdx.x; it < ITEMS; it += THREADS) {
            const int r = it / (COLS / 4), c = 4 * (it % (COLS / 4));
            const int m = m0 + (r >> 5) * SQ + 32 * j + (r & 31), n = n0 + c;
            const bool inside = m < s.M && n < s.n_end;
            if (GATED) {
                const float* p = lds + r * PITCH + (c / (SP / 2)) * SP + c % (SP / 2);
                epi.gated(part, m, n, s.N - n, inside, *reinterpret_cast<const ff_f32x4*>(p), *reinterpret_cast<const ff_f32x4*>(p + SP / 2));
            } else
                epi.plain(part, m, n, s.N - n, inside, *reinterpret_cast<const ff_f32x4*>(lds + r * PITCH + c));
        }
    }
}

// what an output stage reads once a thread: epi.ready(), where it has that
template <typename Epi>
__device__ __forceinline__ auto ff_ready(const Epi& e, int) -> decltype(e.ready()) {
    return e.ready();
}
template <typename Epi>
__device__ __forceinline__ const Epi& ff_ready(const Epi& e, long) {
    return e;
}

// tile BP (rows of P) x BQ (rows of Q), WP x WQ waves
template <typename E, int NP, int BP, int BQ, int WP, int WQ, int BK, bool PO, bool QO, bool GATED, typename Epi>
__global__ void __launch_bounds__(WP* WQ * 64) k_ff_gemm(FfOperand p, FfOperand q, FfShape s, Epi epi) {
    typedef typename FfMfma<E>::V V;
    constexpr int WAVES = WP * WQ, SP = BP / WP, SQ = BQ / WQ, TP = SP / 16, TQ = SQ / 16;
    typedef FfLoader<NP, BP, BK, WAVES, PO, GATED, SP> LP;
    typedef FfLoader<NP, BQ, BK, WAVES, QO, false, SQ> LQ;
    constexpr int BUF = LP::BYTES + LQ::BYTES;
    HIP_DYNAMIC_SHARED(char, lds)
    const int lane = threadIdx.x & 63, wave = ff_wave_index();
    const int wp = wave % WP, wq = wave / WP;
    const int tiles = s.tiles_m * s.tiles_n, part = blockIdx.x / tiles;
    int tm, tn;
    ff_tile_of(s, blockIdx.x - part * tiles, tm, tn);
    const int m0 = tm * BQ, n0 = tn * (GATED ? BP / 2 : BP);
    const int k_lo = part * s.k_part, k_hi = k_lo + s.k_part < s.K ? k_lo + s.k_part : s.K;
    LP lp;
    LQ lq;
    lp.init(p, n0, wave, lane);
    lq.init(q, m0, wave, lane);
    ff_f32x4 acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = ff_f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int LOADS = LP::PER_WAVE + LQ::PER_WAVE;
    auto load_tile = [&](int stage, int k0) {
        lp.load(lds, stage * BUF, k0, k_hi, wave, lane);
        lq.load(lds, stage * BUF + LP::BYTES, k0, k_hi, wave, lane);
    };
    V a[NP][TP], b[2][NP][TQ];
    auto read_p = [&](int at, int i, int kk) {
#pragma unroll
        for (int e = 0; e < NP; ++e) a[e][i] = ff_fragment<V, BP, BK, PO>(lds + at + e * (LP::BYTES / NP), wp * SP + 16 * i, kk, lane);
    };
    auto read_q = [&](int at, int set, int n, int kk) {
        const int e = n / TQ, j = n % TQ;
        b[set][e][j] = ff_fragment<V, BQ, BK, QO>(lds + at + LP::BYTES + e * (LQ::BYTES / NP), wq * SQ + 16 * j, kk, lane);
    };
    if constexpr (NP == 3) {
        // Three planes of a step of 32: three stages of them fill the LDS.  A step waits for its own tile only, with the next one under way, and reads its fragments at
        // its head.
        static_assert(BK == 32, "");
        constexpr int STAGES = 3;
        load_tile(0, k_lo);
        load_tile(1, k_lo + BK);
        int cur = 0, fill = STAGES - 1;
        for (int k0 = k_lo; k0 < k_hi; k0 += BK) {
            ff_dma_barrier<LOADS>();          // the tile has landed for every wave, and the buffer to fill has been read by every wave
            load_tile(fill, k0 + (STAGES - 1) * BK);          // (behind the end the loads go on, from the page of zeros: the count of those under way stays right)
#pragma unroll
            for (int n = 0; n < NP * TQ; ++n) read_q(cur * BUF, 0, n, 0);
#pragma unroll
            for (int i = 0; i < TP; ++i) read_p(cur * BUF, i, 0);
            // smallest products first
#pragma unroll
            for (int o = NP - 1; o >= 0; --o)
#pragma unroll
                for (int e = 0; e <= o; ++e)
#pragma unroll
                    for (int i = 0; i < TP; ++i)
#pragma unroll
                        for (int j = 0; j < TQ; ++j) acc[i][j] = FfMfma<E>::mul(a[e][i], b[0][o - e][j], acc[i][j]);
            cur = cur + 1 == STAGES ? 0 : cur + 1;
            fill = fill + 1 == STAGES ? 0 : fill + 1;
        }
    } else {
        // A step is 64 k (128-byte rows: whole cache lines; with steps of 32 the L2 gave half its rate) in two halves, two stages.  The fragments of a half are read during
        // the half before, each of P's behind its own last product, Q's into a second set: with the first half's products the tile has been read, and one barrier there says
        // both that the next tile has landed and that this one's buffer may be filled again.  The reads and the loads are put between the products by hand:
        // left to itself the compiler gathers the reads in front of their products to save registers, and the matrix pipe waits for them.
        static_assert(BK == 64, "");
        constexpr int PRODUCTS = TP * TQ;
        load_tile(0, k_lo);
        load_tile(1, k_lo + BK);
        ff_dma_barrier<LOADS>();
#pragma unroll
        for (int j = 0; j < TQ; ++j) read_q(0, 0, j, 0);
#pragma unroll
        for (int i = 0; i < TP; ++i) read_p(0, i, 0);
        int cur = 0;
        auto products = [&](auto which, auto whole, int read_at, int load_at, int load_k) {
            constexpr int half = decltype(which)::value, OPS = half == 0 ? TQ : TQ + LOADS;
#pragma unroll
            for (int i = 0; i < TP; ++i)
#pragma unroll
                for (int j = 0; j < TQ; ++j) {
                    const int m = i * TQ + j;
                    acc[i][j] = FfMfma<E>::mul(a[0][i], b[half][0][j], acc[i][j]);
#pragma unroll
                    for (int n = m * OPS / PRODUCTS; n < (m + 1) * OPS / PRODUCTS; ++n) {
                        if (n < TQ) read_q(read_at, half ^ 1, n, half ^ 1);
                        else if (n < TQ + LP::PER_WAVE) lp.template issue<decltype(whole)::value>(n - TQ, lds, load_at, load_k, k_hi, wave, lane);
                        else lq.template issue<decltype(whole)::value>(n - TQ - LP::PER_WAVE, lds, load_at + LP::BYTES, load_k, k_hi, wave, lane);
                    }
                    if (j == TQ - 1) read_p(read_at, i, half ^ 1);
                    ff_keep_order();
                }
        };
        auto step = [&](auto whole, int k0) {
            products(std::integral_constant<int, 0>(), whole, cur * BUF, 0, 0);
            ff_dma_barrier<0>();
            products(std::integral_constant<int, 1>(), whole, (cur ^ 1) * BUF, cur * BUF, k0 + 2 * BK);
            cur ^= 1;
        };
        // two loops, not a choice inside one: the sums of two branches would meet in other registers
        int k0 = k_lo;
        const int k_whole = PO && p.len < k_hi && !(p.len == p.seg && p.len % BK == 0) ? p.len : k_hi;
        for (; k0 + 3 * BK <= k_whole; k0 += BK) step(std::true_type(), k0);
        for (; k0 < k_hi; k0 += BK) step(std::false_type(), k0);
    }
    ff_dma_barrier<0>();          // no load may land in LDS that the workgroup has given back
    ff_output<BP, BQ, WP, WQ, GATED>(reinterpret_cast<float*>(lds), acc, s, m0, n0, part, ff_ready(epi, 0));
}
