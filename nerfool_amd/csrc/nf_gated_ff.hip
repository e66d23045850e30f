// The gated feed-forward block, forward and backward (gnt/transformer_network.py:38-50 is the ungated one: two projections with a ReLU between).
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, out = h Wd^T                                     x [M, D]; Wg, Wu [F, D]; Wd [D, F]
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Forward: one product makes g and u of the same features in one wave's registers and stores h (and, for a backward pass, g and u in float32:
// their rounding to 16 bits would put an error of a bf16 half step into dg and du each, beside the one of dg and du themselves); a second
// makes out.  Backward: dh's product stores [dg | du] (one [M, 2F] tensor) and h again; then dx (k = 2F over [Wg; Wu]), [dWg; dWu] and dWd.
// h, dg and du are rounded once, to the inputs' type, because they are operands of a matrix product in that type.  float32 inputs are split into
// three bf16 parts (8 + 8 + 8 bits, exact) and multiplied as six products of order <= 2^-16: float32-grade sums at 16 / 6 of the float32 pipe's rate.
//
// Bound by the matrix instructions at the clock that the card keeps under them, and by the L2's rate for the tiles.  4096 x 4096 x 8192 bf16: gate and up 442 us (1.24
// PFLOP/s), down 212 us (1.30; a library product of that size 1.45).  4096 x 2048 x 8192, all gradients: forward 281 + 125 + 14 (joining two parts of k), dh and its output
// stage 212, dx 242 + 14, [dWg; dWu] 225, dWd 118.  float32 1500 x 500 x 1333: products of 19 to 38 us, of which about 8 are not the k loop.
#include "nf_ff_gemm.h"
#include "nf_ff_rows.h"

// nf_gated_ff_narrow.hip
bool ff_narrow_fits(int64_t rows, int dim, int hidden);
int64_t ff_narrow_workspace_bytes(int dim, int hidden, int dtype, bool backward);
int ff_narrow(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, int64_t rows, int dim, int hidden, int dtype, int act, void* out, void* workspace,
              hipStream_t st);

namespace {

// ... at p, p + 32, p + 64
__device__ __forceinline__ void ff_put3(ff_bf16* p, int left, const ff_f32x4& v) {
    ff_bf16 t[4][3];
#pragma unroll
    for (int c = 0; c < 4; ++c) ff_split3(c < left ? v[c] : 0.f, t[c]);          // (behind the row's end: zeros)
#pragma unroll
    for (int e = 0; e < 3; ++e) {
        typedef ff_bf16 V4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<V4*>(p + 32 * e) = V4{t[0][e], t[1][e], t[2][e], t[3][e]};
    }
}
// an operand of a later product: 16-bit values, or three planes of bf16 parts (T = float); rows padded to `pitch`, a multiple of ff_pad
template <typename T>
struct FfMid {
    T* p;
    int64_t pitch;
    __device__ __forceinline__ void put(int64_t m, int n, int left, const ff_f32x4& v) const {
        T* d = p + m * pitch + n;
        if (left >= 4) {
            typedef T V4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<V4*>(d) = V4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        } else
            for (int c = 0; c < 4; ++c) d[c] = (T)(c < left ? v[c] : 0.f);
    }
};
template <>
struct FfMid<float> {
    ff_bf16* p;
    int64_t pitch;
    __device__ __forceinline__ void put(int64_t m, int n, int left, const ff_f32x4& v) const { ff_put3(p + 3 * m * pitch + n / 32 * 96 + n % 32, left, v); }
};

template <typename T>
struct EpiStore {
    T *out, *out2;          // nullable
    int64_t pitch;
    int len, split_m;          // rows m < len go to out, rows m >= split_m to out2, at most len of them
    const float* scale;          // [1] times the values (float16 gradients), or null
    float by;
    // (read once a thread, not with every store)
    __device__ __forceinline__ EpiStore ready() const {
        EpiStore e = *this;
        if (std::is_same<T, ff_half>::value) e.by = scale ? scale[1] : 1.f;
        return e;
    }
    __device__ __forceinline__ void plain(int, int m, int n, int left, bool inside, ff_f32x4 v) const {
        if (std::is_same<T, ff_half>::value) v *= by;
        const bool second = m >= split_m;
        const int r = second ? m - split_m : m;
        T* o = second ? out2 : out;
        if (inside && o && r < len) ff_put(o + r * pitch + n, left, v);
    }
    __device__ __forceinline__ void gated(int, int, int, int, bool, const ff_f32x4&, const ff_f32x4&) const {}
};
// a part of the sum over k: [part][M][pitch]
struct EpiPart {
    float* out;
    int64_t pitch, stride;
    __device__ __forceinline__ void plain(int part, int m, int n, int left, bool inside, const ff_f32x4& v) const {
        if (inside) *reinterpret_cast<ff_f32x4*>(out + part * stride + m * pitch + n) = v;          // (pitch is a multiple of 4)
    }
    __device__ __forceinline__ void gated(int, int, int, int, bool, const ff_f32x4&, const ff_f32x4&) const {}
};
template <typename T, bool SIDES>
struct EpiGate {
    FfMid<T> h;
    float *g_save, *u_save;          // [M, F], nullable
    int64_t F;
    int act;
    FfSides sides;
    __device__ __forceinline__ void gated(int, int m, int n, int left, bool inside, ff_f32x4 g, const ff_f32x4& u) const {
        if constexpr (SIDES) ff_sides_settle4<T>(sides, inside, m, n, left, g);
        if (!inside) return;
        ff_f32x4 v;
        float a, slope;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            ff_act(act, g[c], a, slope);
            v[c] = a * u[c];
        }
        h.put(m, n, left, v);
        if (g_save) {
            ff_put(g_save + m * F + n, left, g);
            ff_put(u_save + m * F + n, left, u);
        }
    }
    __device__ __forceinline__ void plain(int, int, int, int, bool, const ff_f32x4&) const {}
};
template <typename T>
struct EpiGateBwd {
    FfMid<T> dgu, h;          // dgu: [M, 2 Fp], dg in columns 0 .., du in columns Fp ..
    const float *g, *u;
    int64_t F, Fp;
    int act, want_h;
    const float* scale;          // float16: [0] times dg and du
    float by;
    __device__ __forceinline__ EpiGateBwd ready() const {
        EpiGateBwd e = *this;
        if (std::is_same<T, ff_half>::value) e.by = scale[0];
        return e;
    }
    __device__ __forceinline__ void plain(int, int m, int n, int left, bool inside, const ff_f32x4& dh) const {
        if (!inside) return;
        ff_f32x4 gv = {0.f, 0.f, 0.f, 0.f}, uv = gv, dg, du, hv;
        const float *gp = g + m * F + n, *up = u + m * F + n;
        if (left >= 4) {
            typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
            gv = *reinterpret_cast<const F4*>(gp);
            uv = *reinterpret_cast<const F4*>(up);
        } else
            for (int c = 0; c < left; ++c) gv[c] = gp[c], uv[c] = up[c];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float a, slope;
            ff_act(act, gv[c], a, slope);
            hv[c] = a * uv[c];
            dg[c] = dh[c] * uv[c] * slope;
            du[c] = dh[c] * a;
            if (std::is_same<T, ff_half>::value) dg[c] *= by, du[c] *= by;
        }
        dgu.put(m, n, left, dg);
        dgu.put(m, (int)Fp + n, left, du);
        if (want_h) h.put(m, n, left, hv);
    }
    __device__ __forceinline__ void gated(int, int, int, int, bool, const ff_f32x4&, const ff_f32x4&) const {}
};

// the parts of a sum over k, added in their order, -> epi
template <typename Epi>
__global__ void __launch_bounds__(256) k_ff_join(EpiPart parts, int n_parts, int64_t M, int N, Epi epi) {
    const int per_row = (int)(parts.pitch / 4);
    const int64_t items = M * per_row;
    const Epi e = epi.ready();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / per_row;
        const int n = (int)(i - m * per_row) * 4;
        const float* p = parts.out + m * parts.pitch + n;
        ff_f32x4 v = *reinterpret_cast<const ff_f32x4*>(p);
        for (int k = 1; k < n_parts; ++k) v += *reinterpret_cast<const ff_f32x4*>(p + k * parts.stride);
        e.plain(0, (int)m, n, N - n, n < N, v);
    }
}

// rows [R, C] -> rows padded with zeros to `pitch`; float -> three planes of bf16 parts.  Up to 5 tensors a launch: blockIdx.y
template <typename T>
struct FfPackJobs {
    struct Job {
        const T* src;
        int64_t rows;
        int cols;
        FfMid<T> dst;
    } job[5];
};
template <typename T>
__global__ void __launch_bounds__(256) k_ff_pack(FfPackJobs<T> jobs) {
    const auto& job = jobs.job[blockIdx.y];
    const int per_row = (int)(job.dst.pitch / 4);
    const int64_t n = job.rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row;
        const int c = (int)(i - r * per_row) * 4, left = job.cols - c;
        ff_f32x4 v;
        const T* s = job.src + r * job.cols + c;
        if (left >= 4) {
            typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            const V4 t = *reinterpret_cast<const V4*>(s);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (float)t[j];
        } else
            for (int j = 0; j < 4; ++j) v[j] = j < left ? (float)s[j] : 0.f;
        job.dst.put(r, c, left > 0 ? left : 0, v);
    }
}

// ---- float16 gradients: the power of two by which dg and du are held (ff_grad_scale), of the largest |dy|.  Two launches; backward pass with all gradients, us without and with them: 40 x
//      2048 x 5504 96 and 104, 64 x 4096 x 8192 204 and 208, 1024 x 1024 x 2048 91 and 98.  (One workgroup for all of a short dy saves 1.5 at 32768 values and loses from 80000 on.)
constexpr int FF_SCALE_PARTS = 256;
__global__ void __launch_bounds__(1024) k_ff_grad_top(const ff_half* __restrict__ dy, int64_t n, float* __restrict__ part) {
    constexpr int N = FfVec<ff_half>::N;
    __shared__ float tops[16];
    float top = 0.f;
    for (int64_t i = ((int64_t)blockIdx.x * 1024 + threadIdx.x) * N; i < n; i += (int64_t)gridDim.x * 1024 * N) {
        float v[N];
        ff_load_row(dy + i, 0, n - i < N ? (int)(n - i) : N, v);
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]));
    }
    top = nf_wave_max(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) top = fmaxf(top, tops[w]);
    if (threadIdx.x == 0) part[blockIdx.x] = top;
}
// out[0] = the scale, out[1] = 1 / it
__global__ void __launch_bounds__(64) k_ff_grad_scale(const float* __restrict__ part, float* __restrict__ out) {
    float top = 0.f;
    for (int i = threadIdx.x; i < FF_SCALE_PARTS; i += 64) top = fmaxf(top, part[i]);
    top = nf_wave_max(top);
    const float s = ff_grad_scale(top);
    if (threadIdx.x == 0) out[0] = s, out[1] = 1.f / s;
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
template <typename T>
struct FfElem {
    typedef T E;
    static constexpr int NP = 1;
};
template <>
struct FfElem<float> {
    typedef ff_bf16 E;
    static constexpr int NP = 3;
};

// rows of operands: 16-byte chunks; three planes lie in blocks of 32
template <typename T>
int64_t ff_pad(int64_t n) {
    return sizeof(T) == 4 ? (n + 31) / 32 * 32 : (n + 7) / 8 * 8;
}

// carves a workspace; with base = nullptr it only counts
struct Carve {
    char* base;
    int64_t used = 0;
    void* take(int64_t bytes) {
        const int64_t at = used;
        used += (bytes + 255) / 256 * 256;
        return base ? base + at : nullptr;
    }
};

template <typename T>
FfMid<T> mid_at(Carve& ws, int64_t rows, int64_t pitch) {
    FfMid<T> m;
    m.p = (T*)ws.take(rows * pitch * sizeof(T));
    m.pitch = pitch;
    return m;
}
template <>
FfMid<float> mid_at<float>(Carve& ws, int64_t rows, int64_t pitch) {
    FfMid<float> m;
    m.p = (ff_bf16*)ws.take(3 * rows * pitch * 2);
    m.pitch = pitch;
    return m;
}
template <typename T>
FfOperand as_operand(const FfMid<T>& m, int rows) {
    return FfOperand{(const uint16_t*)m.p, (const uint16_t*)m.p, m.pitch, rows, 0x7fffffff, 0x7fffffff};
}
FfOperand as_operand(const FfMid<float>& m, int rows) {
    return FfOperand{(const uint16_t*)m.p, (const uint16_t*)m.p, 3 * m.pitch, rows, 0x7fffffff, 0x7fffffff};
}

// a tensor [rows, cols] as an operand: itself where the kernel can read it, else a padded (and for float32 split) copy
template <typename T>
struct FfPacked {
    FfMid<T> mid;
    bool copy;
};
template <typename T>
FfPacked<T> pack_at(Carve& ws, int64_t rows, int cols) {
    FfPacked<T> p;
    p.copy = sizeof(T) == 4 || cols % 8 != 0;
    if (p.copy)
        p.mid = mid_at<T>(ws, rows, ff_pad<T>(cols));
    else {
        p.mid.p = nullptr;
        p.mid.pitch = cols;
    }
    return p;
}
// collects the tensors to copy; those that need no copy are operands as they are
template <typename T>
struct Packing {
    FfPackJobs<T> jobs;
    int n = 0;
    int64_t most = 0;
    void add(const void* src, int64_t rows, int cols, FfPacked<T>& p) {
        if (!p.copy) {
            p.mid.p = (decltype(p.mid.p))const_cast<void*>(src);
            return;
        }
        jobs.job[n++] = {(const T*)src, rows, cols, p.mid};
        const int64_t items = rows * (p.mid.pitch / 4);
        most = items > most ? items : most;
    }
    void run(hipStream_t st) {
        if (!n) return;
        int64_t blocks = (most + 255) / 256;
        if (blocks > 256 * 8) blocks = 256 * 8;
        hipLaunchKernelGGL((k_ff_pack<T>), dim3((unsigned)blocks, n), dim3(256), 0, st, jobs);
    }
};

// steps (of 32) of a part of k: even, as a step of the 16-bit kernel is two of them
int64_t ff_part_steps(int64_t steps, int parts) { return ((steps + parts - 1) / parts + 1) / 2 * 2; }

template <typename E, int NP, int BP, int BQ, int WP, int WQ, int BK, bool PO, bool QO, bool GATED, typename Epi>
int launch(const FfOperand& p, const FfOperand& q, int M, int N, int n_end, int K, int parts, const Epi& epi, hipStream_t st) {
    constexpr int RING = (NP == 3 ? 3 : 2) * NP * (BP + BQ) * BK * 2, OUT = ff_output_bytes<BP, BQ, WP, WQ>(), LDS = RING > OUT ? RING : OUT, COLS = GATED ? BP / 2 : BP;
    static bool set[NF_MAX_DEVICES];
    const int dev = nf_current_device();
    const auto kernel = k_ff_gemm<E, NP, BP, BQ, WP, WQ, BK, PO, QO, GATED, Epi>;
    if (!set[dev]) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            nf_set_error("gated feed-forward: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
            return 2;
        }
        set[dev] = true;
    }
    FfShape s;
    s.M = M, s.N = N, s.K = K, s.n_end = n_end;
    s.tiles_m = (M + BQ - 1) / BQ, s.tiles_n = (N + COLS - 1) / COLS;
    const int steps = (K + BK - 1) / BK;
    s.k_part = ff_part_steps(steps * (BK / 32), parts) * 32;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(s.tiles_m * s.tiles_n * parts)), dim3(WP * WQ * 64), LDS, st, p, q, s, epi);
    return 0;
}

// ---- which tile, and in how many parts k is cut.  The time of a product, in microseconds, as measured on its pieces: a 256 x 256 tile takes 0.85 a k step of 32 and
//      has a CU for itself; two 128 x 128 tiles share one and take 0.7 a step together.  Of a float32 operand's three planes a 128 x 128 tile takes 1.2 a step.  (Tiles of
//      128 x 64 take 0.85 a step: no gain.)  A tile costs about 8 steps beside its k loop (first loads, output stage).  Parts cost their writing and reading, and a launch.
enum { TILE_256, TILE_128, TILE_128_THREE };
struct FfChoice {
    int tile, parts;
};
FfChoice ff_choose(bool three, int64_t M, int64_t N, int64_t K, bool may_split) {
    static const struct {
        int bm, bn, slots;
        double step;
    } tiles[3] = {{256, 256, 256, 0.85}, {128, 128, 512, 0.7}, {128, 128, 256, 1.2}};
    FfChoice best = {three ? TILE_128_THREE : TILE_128, 1};
    double least = 1e30;
    const int64_t steps = (K + 31) / 32;
    for (int tile = three ? TILE_128_THREE : TILE_256; tile <= (three ? TILE_128_THREE : TILE_128); ++tile) {
        const auto& c = tiles[tile];
        const int64_t count = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
        for (int parts = 1; parts <= 8; ++parts) {
            if (parts > 1 && (!may_split || steps < 8 * parts)) break;
            const int64_t per = ff_part_steps(steps, parts), n = count * parts;
            if (per * (parts - 1) >= steps) continue;          // the last part would be empty
            // (a last round that fills less than half of a 128 x 128 tile's slots has the CUs' whole rate for one tile each)
            const int64_t rounds = n / c.slots, rest = n % c.slots;
            double t = rounds * (per + 8) * c.step + (rest ? (per + 8) * c.step * (tile == TILE_128 && rest <= 256 ? 0.6 : 1.0) : 0.0);
            if (parts > 1) t += 4.0 + (double)M * N * 4 * (parts + 1) / 4.5e6;
            if (t < least) least = t, best = {tile, parts};
        }
    }
    return best;
}
int64_t pad4(int64_t n) { return (n + 3) / 4 * 4; }
// ... of each product of the block
enum { FF_GATE_UP, FF_DOWN, FF_DH, FF_DX, FF_DW_GATE_UP, FF_DW_DOWN };
template <typename T>
FfChoice ff_choice_of(int product, int64_t M, int64_t D, int64_t F) {
    const bool three = FfElem<T>::NP == 3;
    const int64_t Dp = ff_pad<T>(D), Fp = ff_pad<T>(F);
    switch (product) {
        case FF_GATE_UP: return ff_choose(three, M, 2 * F, Dp, false);
        case FF_DOWN: return ff_choose(three, M, D, Fp, true);
        case FF_DH: return ff_choose(three, M, F, D, false);
        case FF_DX: return ff_choose(three, M, D, Fp + F, true);
        case FF_DW_GATE_UP: return ff_choose(three, 2 * Fp, D, M, true);
        default: return ff_choose(three, D, F, M, true);
    }
}

// bytes of the parts
int64_t ff_part_bytes(const FfChoice& c, int64_t M, int64_t N) { return c.parts > 1 ? c.parts * M * pad4(N) * 4 : 0; }

template <typename T, bool PO, bool QO, bool GATED, typename Epi>
int product(const FfChoice& c, const FfOperand& p, const FfOperand& q, int M, int N, int n_end, int K, const Epi& epi, hipStream_t st) {
    typedef typename FfElem<T>::E E;
    if constexpr (FfElem<T>::NP == 3) {
        return launch<E, 3, 128, 128, 2, 4, 32, PO, QO, GATED>(p, q, M, N, n_end, K, c.parts, epi, st);
    } else {
        if (c.tile == TILE_256) return launch<E, 1, 256, 256, 2, 4, 64, PO, QO, GATED>(p, q, M, N, n_end, K, c.parts, epi, st);
        return launch<E, 1, 128, 128, 2, 2, 64, PO, QO, GATED>(p, q, M, N, n_end, K, c.parts, epi, st);
    }
}
// ... which may be in parts: `parts` has room for ff_part_bytes
template <typename T, bool PO, bool QO>
int product_split(const FfChoice& c, const FfOperand& p, const FfOperand& q, int M, int N, int K, const EpiStore<T>& epi, float* parts, hipStream_t st) {
    if (c.parts == 1) return product<T, PO, QO, false>(c, p, q, M, N, N, K, epi, st);
    const EpiPart part = {parts, pad4(N), M * pad4(N)};
    const int rc = product<T, PO, QO, false>(c, p, q, M, N, N, K, part, st);
    if (rc) return rc;
    int64_t blocks = (M * (part.pitch / 4) + 255) / 256;
    if (blocks > 256 * 16) blocks = 256 * 16;
    hipLaunchKernelGGL((k_ff_join<EpiStore<T>>), dim3((unsigned)blocks), dim3(256), 0, st, part, c.parts, (int64_t)M, N, epi);
    return 0;
}

#define FF_TRY(call)            \
    do {                        \
        const int rc_ = (call); \
        if (rc_) return rc_;    \
    } while (0)

template <typename T>
struct FwdPlan {
    FfPacked<T> x, wg, wu, wd;
    FfMid<T> h;
    float *parts, *norms;
    int64_t bytes;
    FwdPlan(char* base, int64_t M, int D, int F) {
        Carve ws{base};
        x = pack_at<T>(ws, M, D);
        wg = pack_at<T>(ws, F, D);
        wu = pack_at<T>(ws, F, D);
        wd = pack_at<T>(ws, D, F);
        h = mid_at<T>(ws, M, ff_pad<T>(F));
        parts = (float*)ws.take(ff_part_bytes(ff_choice_of<T>(FF_DOWN, M, D, F), M, D));
        norms = (float*)ws.take((M + F) * 4);
        bytes = ws.used;
    }
};

// Up to this many rows the weights' bytes bound the block and k_ff_rows streams them; above, the tiles of k_ff_gemm read them once for more tokens.  4096 x 8192 bf16, us: 16 rows
// 50 (tiles 87), 48 rows 77 (90), 64 rows 88 (90), 65 rows 131 (90), 128 rows 169 (96); 2048 x 5504 float16: 32 rows 32 (40), 64 rows 45 (42), 65 rows 57 (42).  Short weights and
// float32, whose tiles make six products, would bear more: 520 x 1032 bf16 64 rows 13 (20), 96 rows 14 (21), 128 rows 24 (23); 1024 x 4096 float32 64 rows 36 (87), 128 rows 61 (88).
constexpr int FF_ROWS_MAX = 64;

// ... whose h begins the workspace
int64_t ff_few_rows_h_bytes(int64_t M, int F, int value_bytes) { return (M * F * value_bytes + 255) / 256 * 256; }

template <typename T, bool GATED, bool SIDES>
int few_rows(const void* w0, const void* w1, const void* x, int M, int N, int K, void* out, float* g_save, float* u_save, int act, const FfSides& sides, hipStream_t st) {
    switch (ff_rows_tokens(M, (N + 15) / 16)) {
        case 1: return ff_rows_launch<T, 1, GATED, SIDES>(w0, w1, x, M, N, K, out, g_save, u_save, act, sides, st);
        case 2: return ff_rows_launch<T, 2, GATED, SIDES>(w0, w1, x, M, N, K, out, g_save, u_save, act, sides, st);
        case 3: return ff_rows_launch<T, 3, GATED, SIDES>(w0, w1, x, M, N, K, out, g_save, u_save, act, sides, st);
        default: return ff_rows_launch<T, 4, GATED, SIDES>(w0, w1, x, M, N, K, out, g_save, u_save, act, sides, st);
    }
}

template <typename T>
int ff_fwd(const void* x, const void* wg, const void* wu, const void* wd, int M, int D, int F, int act, void* out, float* g_save, float* u_save,
           void* workspace, hipStream_t st) {
    // relu's sides are asked for by a backward pass only
    const bool border = act == FF_RELU && g_save;
    FfSides sides = {};
    if (M <= FF_ROWS_MAX) {
        if (border) {
            sides = ff_sides<T>(x, wg, M, F, D, sizeof(T) == 4 ? D / 4 : D / 32, (float*)((char*)workspace + ff_few_rows_h_bytes(M, F, sizeof(T))), st);
            FF_TRY((few_rows<T, true, true>(wg, wu, x, M, F, D, workspace, g_save, u_save, act, sides, st)));
        } else
            FF_TRY((few_rows<T, true, false>(wg, wu, x, M, F, D, workspace, g_save, u_save, act, sides, st)));
        return few_rows<T, false, false>(wd, nullptr, workspace, M, D, F, out, nullptr, nullptr, 0, sides, st);
    }
    FwdPlan<T> f((char*)workspace, M, D, F);
    if (border) sides = ff_sides<T>(x, wg, M, F, D, FfElem<T>::NP == 3 ? 6 * D / 32 : D / 32, f.norms, st);
    Packing<T> pack;
    pack.add(x, M, D, f.x);
    pack.add(wg, F, D, f.wg);
    pack.add(wu, F, D, f.wu);
    pack.add(wd, D, F, f.wd);
    pack.run(st);
    FfOperand p = as_operand(f.wg.mid, F);
    p.b = (const uint16_t*)f.wu.mid.p;
    const FfOperand q = as_operand(f.x.mid, M);
    const FfChoice c = ff_choice_of<T>(FF_GATE_UP, M, D, F);
    if (border) FF_TRY((product<T, false, false, true>(c, p, q, M, F, (int)f.h.pitch, (int)f.x.mid.pitch, EpiGate<T, true>{f.h, g_save, u_save, F, act, sides}, st)));
    else FF_TRY((product<T, false, false, true>(c, p, q, M, F, (int)f.h.pitch, (int)f.x.mid.pitch, EpiGate<T, false>{f.h, g_save, u_save, F, act, sides}, st)));
    const EpiStore<T> store = {(T*)out, nullptr, D, M, 0x7fffffff, nullptr, 1.f};
    FF_TRY((product_split<T, false, false>(ff_choice_of<T>(FF_DOWN, M, D, F), as_operand(f.wd.mid, D), as_operand(f.h, M), M, D, (int)f.h.pitch, store, f.parts, st)));
    return 0;
}

template <typename T>
struct BwdPlan {
    FfPacked<T> x, wg, wu, wd, dy;
    FfMid<T> dgu, h;
    float* parts;          // of one product at a time
    float* scale;          // float16
    int64_t bytes;
    BwdPlan(char* base, int64_t M, int D, int F, bool dx, bool dwgu, bool dwd) {
        Carve ws{base};
        dy = pack_at<T>(ws, M, D);
        wd = pack_at<T>(ws, D, F);
        if (dwgu) x = pack_at<T>(ws, M, D);
        if (dx) wg = pack_at<T>(ws, F, D), wu = pack_at<T>(ws, F, D);
        dgu = mid_at<T>(ws, M, 2 * ff_pad<T>(F));
        if (dwd) h = mid_at<T>(ws, M, ff_pad<T>(F));
        int64_t most = 0;
        const auto room = [&](int product, int64_t rows, int64_t cols) {
            const int64_t n = ff_part_bytes(ff_choice_of<T>(product, M, D, F), rows, cols);
            most = n > most ? n : most;
        };
        if (dx) room(FF_DX, M, D);
        if (dwgu) room(FF_DW_GATE_UP, 2 * ff_pad<T>(F), D);
        if (dwd) room(FF_DW_DOWN, D, F);
        parts = (float*)ws.take(most);
        scale = (float*)ws.take(sizeof(T) == 2 ? (2 + FF_SCALE_PARTS) * 4 : 0);
        bytes = ws.used;
    }
};

template <typename T>
int ff_bwd(const void* x, const void* wg, const void* wu, const void* wd, const void* dy, const float* g, const float* u, int M, int D, int F,
           int act, void* dx, void* dwg, void* dwu, void* dwd, void* workspace, hipStream_t st) {
    const bool dwgu = dwg || dwu;
    BwdPlan<T> f((char*)workspace, M, D, F, dx != nullptr, dwgu, dwd != nullptr);
    const int Fp = (int)ff_pad<T>(F);
    Packing<T> pack;
    pack.add(dy, M, D, f.dy);
    pack.add(wd, D, F, f.wd);
    if (dx) {
        pack.add(wg, F, D, f.wg);
        pack.add(wu, F, D, f.wu);
    }
    if (dwgu) pack.add(x, M, D, f.x);
    pack.run(st);
    // dh[m][f] = sum over d of dy[m][d] Wd[d][f]
    const float* scale = nullptr;
    if (std::is_same<T, ff_half>::value) {
        hipLaunchKernelGGL(k_ff_grad_top, dim3(FF_SCALE_PARTS), dim3(1024), 0, st, (const ff_half*)dy, (int64_t)M * D, f.scale + 2);
        hipLaunchKernelGGL(k_ff_grad_scale, dim3(1), dim3(64), 0, st, (const float*)f.scale + 2, f.scale);
        scale = f.scale;
    }
    const EpiGateBwd<T> gate = {f.dgu, f.h, g, u, F, Fp, act, dwd != nullptr, scale, 1.f};
    FfOperand p = as_operand(f.wd.mid, (int)f.wd.mid.pitch);
    FF_TRY((product<T, true, false, false>(ff_choice_of<T>(FF_DH, M, D, F), p, as_operand(f.dy.mid, M), M, F, Fp, D, gate, st)));
    if (dx) {          // dx[m][d] = sum over k of dgu[m][k] [Wg; zeros up to Fp; Wu][k][d]
        p = as_operand(f.wg.mid, (int)f.wg.mid.pitch);
        p.b = (const uint16_t*)f.wu.mid.p;
        p.len = F, p.seg = Fp;
        const EpiStore<T> store = {(T*)dx, nullptr, D, M, 0x7fffffff, scale, 1.f};
        FF_TRY((product_split<T, true, false>(ff_choice_of<T>(FF_DX, M, D, F), p, as_operand(f.dgu, M), M, D, Fp + F, store, f.parts, st)));
    }
    if (dwgu) {          // [dWg; dWu][f][d] = sum over m of dgu[m][f] x[m][d]
        const EpiStore<T> store = {(T*)dwg, (T*)dwu, D, F, Fp, scale, 1.f};
        FF_TRY((product_split<T, true, true>(ff_choice_of<T>(FF_DW_GATE_UP, M, D, F), as_operand(f.x.mid, (int)f.x.mid.pitch), as_operand(f.dgu, 2 * Fp), 2 * Fp, D, M, store,
                                                  f.parts, st)));
    }
    if (dwd) {          // dWd[d][f] = sum over m of dy[m][d] h[m][f]
        const EpiStore<T> store = {(T*)dwd, nullptr, F, D, 0x7fffffff, nullptr, 1.f};
        FF_TRY((product_split<T, true, true>(ff_choice_of<T>(FF_DW_DOWN, M, D, F), as_operand(f.h, Fp), as_operand(f.dy.mid, (int)f.dy.mid.pitch), D, F, M, store, f.parts,
                                                  st)));
    }
    return 0;
}

bool ff_sizes_ok(const char* what, int64_t M, int D, int F, int dtype, int act) {
    if (M >= 1 && M <= (1 << 30) && D >= 1 && F >= 1 && D <= (1 << 20) && F <= (1 << 20) && dtype >= FF_F32 && dtype <= FF_F16 && act >= FF_SILU && act <= FF_RELU)
        return true;
    nf_set_error("%s: need 1 <= rows <= 2^30, 1 <= dim, hidden <= 2^20, dtype and activation in 0 .. 2 (got rows %lld dim %d hidden %d dtype %d activation %d)",
                 what, (long long)M, D, F, dtype, act);
    return false;
}

}  // namespace

extern "C" int64_t nf_gated_ff_fwd_workspace_bytes(int64_t rows, int dim, int hidden, int dtype) {
    if (!ff_sizes_ok("nf_gated_ff_fwd_workspace_bytes", rows, dim, hidden, dtype, 0)) return -1;
    if (rows <= FF_ROWS_MAX) return ff_few_rows_h_bytes(rows, hidden, dtype == FF_F32 ? 4 : 2) + (rows + hidden) * 4;
    const int64_t n = dtype == FF_F32 ? FwdPlan<float>(nullptr, rows, dim, hidden).bytes : FwdPlan<ff_bf16>(nullptr, rows, dim, hidden).bytes;
    const int64_t narrow = ff_narrow_fits(rows, dim, hidden) ? ff_narrow_workspace_bytes(dim, hidden, dtype, false) : 0;
    return n > narrow ? n : narrow;          // (which of the two runs depends on whether g and u are saved)
}

extern "C" int nf_gated_ff_fwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, int64_t rows, int dim, int hidden, int dtype,
                               int activation, void* out, float* g_save, float* u_save, void* workspace, nf_stream_t stream) {
    if (!ff_sizes_ok("nf_gated_ff_fwd", rows, dim, hidden, dtype, activation)) return 1;
    NF_REQUIRE((g_save != nullptr) == (u_save != nullptr), "nf_gated_ff_fwd: g_save and u_save go together");
    if (rows > FF_ROWS_MAX && !g_save && ff_narrow_fits(rows, dim, hidden)) {
        FF_TRY(ff_narrow(x, w_gate, w_up, w_down, nullptr, rows, dim, hidden, dtype, activation, out, workspace, (hipStream_t)stream));
        NF_LAUNCH_CHECK("nf_gated_ff_fwd");
        return 0;
    }
    const auto f = dtype == FF_F32 ? ff_fwd<float> : dtype == FF_BF16 ? ff_fwd<ff_bf16> : ff_fwd<ff_half>;
    FF_TRY(f(x, w_gate, w_up, w_down, (int)rows, dim, hidden, activation, out, g_save, u_save, workspace, (hipStream_t)stream));
    NF_LAUNCH_CHECK("nf_gated_ff_fwd");
    return 0;
}

extern "C" int nf_gated_ff_bwd_recomputes(int64_t rows, int dim, int hidden) { return ff_narrow_fits(rows, dim, hidden); }

extern "C" int64_t nf_gated_ff_bwd_workspace_bytes(int64_t rows, int dim, int hidden, int dtype, int want_dx, int want_dw_gate_up, int want_dw_down) {
    if (!ff_sizes_ok("nf_gated_ff_bwd_workspace_bytes", rows, dim, hidden, dtype, 0)) return -1;
    if (want_dx && !want_dw_gate_up && !want_dw_down && ff_narrow_fits(rows, dim, hidden)) return ff_narrow_workspace_bytes(dim, hidden, dtype, true);
    if (dtype == FF_F32) return BwdPlan<float>(nullptr, rows, dim, hidden, want_dx, want_dw_gate_up, want_dw_down).bytes;
    return BwdPlan<ff_bf16>(nullptr, rows, dim, hidden, want_dx, want_dw_gate_up, want_dw_down).bytes;
}

extern "C" int nf_gated_ff_bwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, const void* dy, const float* g, const float* u,
                               int64_t rows, int dim, int hidden, int dtype, int activation, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                               void* workspace, nf_stream_t stream) {
    if (!ff_sizes_ok("nf_gated_ff_bwd", rows, dim, hidden, dtype, activation)) return 1;
    if (dx && !dw_gate && !dw_up && !dw_down && ff_narrow_fits(rows, dim, hidden)) {
        FF_TRY(ff_narrow(x, w_gate, w_up, w_down, dy, rows, dim, hidden, dtype, activation, dx, workspace, (hipStream_t)stream));
        NF_LAUNCH_CHECK("nf_gated_ff_bwd");
        return 0;
    }
    NF_REQUIRE(g && u, "nf_gated_ff_bwd: these sizes and gradients need the forward's g and u");
    const auto f = dtype == FF_F32 ? ff_bwd<float> : dtype == FF_BF16 ? ff_bwd<ff_bf16> : ff_bwd<ff_half>;
    FF_TRY(f(x, w_gate, w_up, w_down, dy, g, u, (int)rows, dim, hidden, activation, dx, dw_gate, dw_up, dw_down, workspace, (hipStream_t)stream));
    NF_LAUNCH_CHECK("nf_gated_ff_bwd");
    return 0;
}

extern "C" int nf_gated_ff_form(int64_t rows, int dim, int hidden, int dtype, int product) {
    if (!ff_sizes_ok("nf_gated_ff_form", rows, dim, hidden, dtype, 0)) return -1;
    if (product < 0 || product > 5) {
        nf_set_error("nf_gated_ff_form: product in 0 .. 5 (got %d)", product);
        return -1;
    }
    if (product <= FF_DOWN && rows <= FF_ROWS_MAX) return 0;
    const FfChoice c = dtype == FF_F32 ? ff_choice_of<float>(product, rows, dim, hidden) : ff_choice_of<ff_bf16>(product, rows, dim, hidden);
    return c.parts << 16 | (c.tile == TILE_256 ? 256 : 128);
}
