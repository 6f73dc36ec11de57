// Token-major matrix product with a fused epilogue: y = act(x W^T + b) + r.
//   x (M,C) rows, W (K,C) rows, b (K) float32, r and y (M,K) rows; float32, float16 or bfloat16 storage, products and the
//   sum over C in float32 on the matrix cores, epilogue in float32, one rounding at the store.
//
// Two forms, chosen by plan():
//   tiles   a workgroup forms a BM x BN tile of y; both operands go through LDS in slabs of 128 bytes per row.  Bound by the matrix
//           cores, in practice by the chip's power: 16384 x 4096 x 16384 bfloat16 with GELU 1.84 ms = 1.20 PFLOP/s (matrix cores
//           busy 57 %), 8191 x 8192 x 4096 float16 0.45 ms = 1.23 PFLOP/s (62 %).  With some tens of rows bound by the read
//           of W: 37 x 4096 x 16384 33 us = 4.1 TB/s.
//   rows    up to 16 rows of x: waves stream W from memory into registers.  One row of 4096 x 4096: 9.9 us on the device, of
//           which 6.9 are the read of W at a large copy's rate.
// Both can be split over C: partial sums go to a workspace and a second kernel adds them in a fixed order.
#include "vo_tokens.h"

namespace {

struct LinArgs {
    const void* x;
    const void* w;
    const float* bias;
    const void* res;
    void* y;
    float* part;                     // split over C: partial sums (splits, M, K)
    int64_t xs, rs, ys;              // row strides in elements
    int64_t M;
    int C, K, act;
    int splits, c_per_split;         // c_per_split: a multiple of the slab
    unsigned tiles_m, tiles_n;
};

// z / (1 + e^-u): the exponential is exp2 of u log2(e), rounded once, so its relative error grows like |u| 2^-24; where |u| is
// large the sum is 1 or the quotient has vanished from 16 bits.  float32 storage takes the library's functions.
template <bool EXACT> __device__ __forceinline__ float over_sigmoid(float z, float u) {
    if constexpr (EXACT) return z / (1.f + expf(-u));
    return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * u));
}

// GELU is max(z, 0) - |z| Q(|z|), Q(u) = erfc(u / sqrt 2) / 2: below zero nothing is subtracted, so the result keeps its digits however
// small it is (0.5 z (1 + erf) has lost half of them by z = -3 and all by -6).  For results of 16 bits
// Q(u) = e^(-u^2 / 2) P(t), t = 1 / (1 + 0.36 u), P fitted for the least relative error (8e-7) over u = 0 to 13.5, where Q leaves
// float32.  (The library's functions take several branches in most waves: with erff GELU's share of a 16384 x 4096 x 16384 product was
// 150 us of 1883.)
__device__ __forceinline__ float gelu_short(float z) {
    const float u = fabsf(fminf(z, 30.f)), t = __builtin_amdgcn_rcpf(1.f + 0.36f * u);        // +infinity stays, with no 0 times it
    const float p = t * (0.143717435f + t * (0.141710669f + t * (0.140057433f + t * (0.0256238089f + t * (0.1822976f + t * (-0.180751654f + t * 0.0473445675f))))));
    return (z < 0.f ? 0.f : z) - u * p * __builtin_amdgcn_exp2f(-0.721347520444481703f * u * u);
}

template <bool EXACT> __device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case VO_ACT_RELU: return z < 0.f ? 0.f : z;                                          // NaN stays NaN
        case VO_ACT_GELU: return EXACT ? 0.5f * z * erfcf(z * -0.70710678118654752f) : gelu_short(z);
        case VO_ACT_GELU_TANH:                                                               // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
            return over_sigmoid<EXACT>(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
        case VO_ACT_SILU: return over_sigmoid<EXACT>(z, z);
        default: return z;
    }
}

// PER consecutive outputs k.. of one row: the bias and the residual are fetched ahead of their use.  A row's last, shorter
// piece goes element by element.
template <typename T> struct Piece {
    static constexpr int PER = vo_elem<T>::PER;
    vo_u32x4 res;

    static __device__ __forceinline__ void load_bias(const LinArgs& a, int k, float* bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j) bias[j] = a.bias && k + j < a.K ? a.bias[k + j] : 0.f;
    }
    __device__ __forceinline__ void load_residual(const LinArgs& a, int64_t m, int k) {
        res = vo_u32x4{0, 0, 0, 0};
        if (a.res && m < a.M && k + PER <= a.K) res = vo_load16(static_cast<const T*>(a.res) + m * a.rs + k);
    }
    // bias, activation, residual, one rounding
    __device__ __forceinline__ void finish(const LinArgs& a, int64_t m, int k, const float* acc, const float* bias) const {
        T* y = static_cast<T*>(a.y) + m * a.ys + k;
        float v[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = activate<sizeof(T) == 4>(acc[j] + bias[j], a.act);
        if (k + PER <= a.K) {
            if (a.res) {
                float r[PER];
                vo_elem<T>::unpack(res, r);
#pragma unroll
                for (int j = 0; j < PER; ++j) v[j] += r[j];
            }
            vo_store16(y, vo_elem<T>::pack(v));
        } else {
            const T* r = static_cast<const T*>(a.res) + m * a.rs + k;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (k + j < a.K) vo_elem<T>::put(y + j, v[j] + (a.res ? vo_elem<T>::get(r + j) : 0.f));
        }
    }
    // into the workspace or through the epilogue
    __device__ __forceinline__ void emit(const LinArgs& a, int split, int64_t m, int k, const float* acc, const float* bias) const {
        if (a.splits > 1) {
            float* p = a.part + ((int64_t)split * a.M + m) * a.K + k;
            if (k + PER <= a.K) {
#pragma unroll
                for (int j = 0; j < PER; j += 4) vo_store16(p + j, __builtin_bit_cast(vo_u32x4, vo_f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]}));
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j)
                    if (k + j < a.K) p[j] = acc[j];
            }
        } else {
            finish(a, m, k, acc, bias);
        }
    }
};

// ------------------------------------------------------------------------------------------------------------ tiles
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// WGM x WGN waves; a wave owns TM rows of x times TN outputs as 16x16 products with W as the first operand, so that a lane
// holds four consecutive outputs of one row.  LDS rows are 128 bytes (eight chunks); chunk c of row r sits at
// c ^ (r / 2 % 8), which spreads the 16-byte reads of sixteen rows over all 64 banks (r % 8 in its place: half of the LDS cycles
// were conflicts).  The permutation is applied to the addresses the lanes
// fetch, because a load into LDS places lane l's bytes at position l.
template <typename T, int BM, int BN, int WGM, int WGN, int STAGES, bool DIRECT>
__global__ __launch_bounds__(64 * WGM * WGN) void linear_tiles(const LinArgs a) {
    constexpr int PER = vo_elem<T>::PER, BK = 8 * PER, NW = WGM * WGN;
    constexpr int TM = BM / WGM, TN = BN / WGN, MT = TM / 16, NT = TN / 16;
    constexpr int ROWS = BM + BN, LOADS = ROWS / 8 / NW;             // 1 KiB wave loads (8 rows) per wave and slab
    constexpr int STRIP = TN + 4;                                    // floats per row of the store's staging strip
    constexpr int SLAB = ROWS * 128, STAGE = NW * 16 * STRIP * 4;
    static_assert(ROWS % (8 * NW) == 0 && BM % (8 * NW) == 0, "a wave's loads must not straddle the operands");
    static_assert(DIRECT || STAGES == 2, "registers hold two more slabs");
    __shared__ __align__(16) unsigned char lds[STAGES * SLAB > STAGE ? STAGES * SLAB : STAGE];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // tile order: splits outermost, then bands of 8 row tiles, within a band column by column
    const unsigned per_split = a.tiles_m * a.tiles_n;
    unsigned id = vo_xcd_contiguous(blockIdx.x, per_split * a.splits);
    const int split = id / per_split;
    id %= per_split;
    const unsigned band = id / (8 * a.tiles_n), in_band = id % (8 * a.tiles_n);
    const unsigned band_rows = a.tiles_m - band * 8 < 8 ? a.tiles_m - band * 8 : 8;
    const int64_t m0 = (int64_t)(band * 8 + in_band % band_rows) * BM;
    const int n0 = (int)(in_band / band_rows) * BN;
    const int c_first = split * a.c_per_split;
    const int c_last = a.C - c_first < a.c_per_split ? a.C : c_first + a.c_per_split;
    const int slabs = (c_last - c_first + BK - 1) / BK;

    const int64_t xb = (int64_t)sizeof(T) * a.xs, wb = (int64_t)sizeof(T) * a.C;
    const int rows_x = (int)(a.M - m0 < BM ? a.M - m0 : BM), rows_w = a.K - n0 < BN ? a.K - n0 : BN;
    const T* xt = static_cast<const T*>(a.x) + m0 * a.xs;
    const T* wt = static_cast<const T*>(a.w) + (int64_t)n0 * a.C;
    const __amdgpu_buffer_rsrc_t xrs = vo_buffer(xt, (rows_x - 1) * xb + wb);
    const __amdgpu_buffer_rsrc_t wrs = vo_buffer(wt, rows_w * wb);

    constexpr int XL = LOADS * BM / ROWS;                            // loads 0 .. XL - 1 of a wave fetch x, the rest W
    const int sub = lane >> 3;                                       // this lane's row of a load's eight
    auto is_x = [&](int i) { return i < XL; };
    auto tile_row = [&](int i) {                                     // first of the eight rows of load i, within its operand
        return (is_x(i) ? wave * XL + i : wave * (LOADS - XL) + i - XL) * 8;
    };
    auto chunk = [&](int i) { return (lane & 7) ^ swizzle(tile_row(i) + sub); };             // the chunk it fetches
    // Offsets of an operand's first two loads (the chunk order repeats every 16 rows); load i lies i whole loads further.  Rows
    // behind the operand's last lie behind its descriptor and become zero by themselves.
    unsigned first[2][2];
    int ahead_of[2][2];                                              // elements of C ahead of the chunk within the slab
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int i = o == 0 ? q : XL + q;
            first[o][q] = (unsigned)((tile_row(i) - q * 8 + sub) * (o == 0 ? xb : wb)) + chunk(i) * 16;
            ahead_of[o][q] = chunk(i) * PER;
        }
    struct Regs { vo_u32x4 r[DIRECT ? 1 : LOADS]; };                 // unaligned rows pass through registers
    auto fetch = [&](int s, unsigned char* buf, Regs& regs) {
        const int c0 = c_first + s * BK;
        if constexpr (DIRECT) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {                        // whole chunks: C is a multiple of PER
                const int o = is_x(i) ? 0 : 1, j = is_x(i) ? i : i - XL;
                const unsigned at = first[o][j & 1] + (unsigned)(c0 * (int)sizeof(T) + j * 8 * (int)(o == 0 ? xb : wb));
                vo_load_to_lds(o == 0 ? xrs : wrs, buf + (o == 0 ? 0 : BM * 128) + tile_row(i) * 128,
                               ahead_of[o][j & 1] < c_last - c0 ? at : VO_OUTSIDE);
            }
        } else if (a.C >= PER) {
            // a row's last, shorter piece is fetched as the row's last 16 bytes and moved down when it is put into LDS
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = tile_row(i) + sub, c = c0 + chunk(i) * PER, gone = c + PER > c_last ? c + PER - c_last : 0;
                regs.r[i] = vo_u32x4{0, 0, 0, 0};
                if (gone < PER && r < (is_x(i) ? rows_x : rows_w))
                    regs.r[i] = vo_load16((is_x(i) ? xt + r * a.xs : wt + (int64_t)r * a.C) + c - gone);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = tile_row(i) + sub, c = c0 + chunk(i) * PER;
                const T* p = (is_x(i) ? xt + r * a.xs : wt + (int64_t)r * a.C) + c;
                regs.r[i] = vo_load_unaligned<T>(p, r < (is_x(i) ? rows_x : rows_w) ? c_last - c : 0, c);
            }
        }
    };
    auto put = [&](int s, unsigned char* buf, Regs& regs) {
        if constexpr (!DIRECT) {
            const int c0 = c_first + s * BK;
            if (c0 + BK > c_last && a.C >= PER) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int gone = c0 + chunk(i) * PER + PER - c_last;
                    if (gone > 0 && gone < PER) regs.r[i] = vo_move_down(regs.r[i], gone * (int)sizeof(T));
                }
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                *reinterpret_cast<vo_u32x4*>(buf + (is_x(i) ? 0 : BM * 128) + tile_row(i) * 128 + lane * 16) = regs.r[i];
        }
    };

    const int wm = wave / WGN, wn = wave % WGN;
    vo_f32x4 acc[NT][MT] = {};
    const int fr = lane & 15, fg = lane >> 4;
    struct Frags { vo_u32x4 w[NT], x[MT]; } f0, f1;                  // operands of 64 bytes of the rows
    auto read = [&](Frags& f, const unsigned char* buf, int part) {
        const int pos = ((part * 4 + fg) ^ swizzle(fr)) * 16;
#pragma unroll
        for (int i = 0; i < NT; ++i) f.w[i] = *reinterpret_cast<const vo_u32x4*>(buf + (BM + wn * TN + i * 16 + fr) * 128 + pos);
#pragma unroll
        for (int i = 0; i < MT; ++i) f.x[i] = *reinterpret_cast<const vo_u32x4*>(buf + (wm * TM + i * 16 + fr) * 128 + pos);
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int part = 0; part < vo_elem<T>::PARTS; ++part)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = vo_elem<T>::mma16(f.w[i], f.x[j], acc[i][j], part);
    };
    // one LDS read per few products, so that neither pipe waits for the other
    auto interleave = [&]() {
        constexpr int PRODUCTS = NT * MT * vo_elem<T>::PARTS, READS = NT + MT, EACH = PRODUCTS / READS > 0 ? PRODUCTS / READS : 1;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        }
        if constexpr (PRODUCTS > READS * EACH) __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS - READS * EACH, 0);
    };

    // While one half of a slab is multiplied the operands of the next half are read from LDS.  The barrier sits between the
    // halves: there slab s has been read to its end by all waves (its buffer takes slab s + STAGES) and slab s + 1 has
    // arrived; the loads of the slabs behind that stay under way.  Slabs past the end are fetched too (as zeros, without
    // any traffic), so that the number of loads under way is always the same.
    unsigned char* buf = lds;                                        // of slab s
    auto after = [&](unsigned char* p) { return p + SLAB == lds + STAGES * SLAB ? lds : p + SLAB; };
    Regs even, odd;                                                  // slabs on their way through registers
    auto step = [&](int s, Regs& regs) {                             // regs: slab s + 2
        read(f1, buf, 1);
        multiply(f0);
        interleave();
        if constexpr (DIRECT) {
            vo_lds_barrier<(STAGES - 2) * LOADS>();
            fetch(s + STAGES, buf, regs);
        } else {
            __syncthreads();
            if (s + 2 < slabs) put(s + 2, buf, regs);
            if (s + 4 < slabs) fetch(s + 4, nullptr, regs);
        }
        buf = after(buf);
        read(f0, buf, 0);
        multiply(f1);
        interleave();
    };
    if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) fetch(i, lds + i * SLAB, even);
        vo_lds_barrier<(STAGES - 1) * LOADS>();
        read(f0, buf, 0);
        for (int s = 0; s + 1 < slabs; ++s) step(s, even);
    } else {
        fetch(0, nullptr, even);
        if (slabs > 1) fetch(1, nullptr, odd);
        put(0, lds, even);
        if (slabs > 2) fetch(2, nullptr, even);
        if (slabs > 1) put(1, lds + SLAB, odd);
        if (slabs > 3) fetch(3, nullptr, odd);
        __syncthreads();
        read(f0, buf, 0);
        int s = 0;
        for (; s + 2 < slabs; s += 2) {
            step(s, even);
            step(s + 1, odd);
        }
        if (s + 1 < slabs) step(s, even);
    }
    read(f1, buf, 1);
    multiply(f0);
    interleave();
    multiply(f1);

    // store: sixteen rows at a time through a strip of LDS of the wave's own, so that rows leave in 16-byte pieces.  The
    // loop stays rolled (the epilogue's code is long) and the sums move down one place per round, because a register
    // array with a running index would live in memory.  The residual's pieces are fetched a round ahead.
    float* strip = reinterpret_cast<float*>(lds) + wave * 16 * STRIP;
    constexpr int ACROSS = TN / PER, PIECES = 16 * ACROSS >= 64 ? 16 * ACROSS / 64 : 1;   // 16-byte pieces per row; per lane and round
    static_assert(64 % ACROSS == 0, "a lane keeps to its columns");
    const int col = lane % ACROSS * PER, k = n0 + wn * TN + col;
    const int64_t m_first = m0 + wm * TM + lane / ACROSS;
    constexpr int STEP = 64 / ACROSS;                                // rows between a lane's pieces
    float bias[PER];
    Piece<T> ahead[PIECES];
    Piece<T>::load_bias(a, k, bias);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) ahead[p].load_residual(a, m_first + p * STEP, k);
    vo_lds_barrier();
#pragma unroll 1
    for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int i = 0; i < NT; ++i) *reinterpret_cast<vo_f32x4*>(strip + fr * STRIP + i * 16 + fg * 4) = acc[i][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int q = 0; q + 1 < MT; ++q) acc[i][q] = acc[i][q + 1];
        Piece<T> now[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            now[p] = ahead[p];
            if (j + 1 < MT) ahead[p].load_residual(a, m_first + (j + 1) * 16 + p * STEP, k);
        }
        vo_wave_lds_fence();
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int64_t m = m_first + j * 16 + p * STEP;
            if (m < a.M && k < a.K && lane / ACROSS + p * STEP < 16) {
                float v[PER];
#pragma unroll
                for (int q = 0; q < PER; q += 4) {
                    const vo_f32x4 t = *reinterpret_cast<const vo_f32x4*>(strip + (lane / ACROSS + p * STEP) * STRIP + col + q);
                    v[q] = t[0]; v[q + 1] = t[1]; v[q + 2] = t[2]; v[q + 3] = t[3];
                }
                now[p].emit(a, split, m, k, v, bias);
            }
        }
        vo_wave_lds_fence();
    }
}

// ------------------------------------------------------------------------------------------------------------- rows
// At most 16 rows of x: a workgroup forms 16 outputs for all of them, its eight waves each a part of C; W goes from memory
// to registers once, the rows of x come from the caches.  The waves' sums are added in LDS in wave order.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(512) void linear_rows(const LinArgs a) {
    constexpr int PER = vo_elem<T>::PER, STEP = 4 * PER, NW = 8;     // one product covers STEP elements of C
    __shared__ __align__(16) float sums[NW][16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const unsigned id = vo_xcd_contiguous(blockIdx.x, a.tiles_n * a.splits);
    const int split = id / a.tiles_n, n0 = (int)(id % a.tiles_n) * 16;
    const int c_first = split * a.c_per_split;
    const int c_last = a.C - c_first < a.c_per_split ? a.C : c_first + a.c_per_split;
    // parts of whole pairs of steps: 128 bytes of a row of W
    const int part = ((c_last - c_first + 2 * STEP - 1) / (2 * STEP) + NW - 1) / NW * 2 * STEP;
    const int c_lo = c_first + wave * part < c_last ? c_first + wave * part : c_last;
    const int c_hi = c_lo + part < c_last ? c_lo + part : c_last;

    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.w) + (int64_t)n0 * a.C;
    const int64_t xb = (int64_t)sizeof(T) * a.xs, wb = (int64_t)sizeof(T) * a.C;
    const int rows_w = a.K - n0 < 16 ? a.K - n0 : 16;
    const __amdgpu_buffer_rsrc_t xrs = vo_buffer(x, (a.M - 1) * xb + wb);
    const __amdgpu_buffer_rsrc_t wrs = vo_buffer(w, rows_w * wb);
    const unsigned xo = fr < a.M ? (unsigned)(fr * xb) + fg * 16 : VO_OUTSIDE;
    const unsigned wo = fr < rows_w ? (unsigned)(fr * wb) + fg * 16 : VO_OUTSIDE;

    constexpr int DEPTH = 8;                                         // steps whose loads are issued together
    vo_f32x4 acc = {};
    for (int first = c_lo; first < c_hi; first += DEPTH * STEP) {
        vo_u32x4 wf[DEPTH], xf[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int c = first + d * STEP + fg * PER;
            if constexpr (ALIGNED) {
                const unsigned at = (first + d * STEP) * (unsigned)sizeof(T);
                wf[d] = __builtin_amdgcn_raw_buffer_load_b128(wrs, c < c_hi ? wo + at : VO_OUTSIDE, 0, 0);
                xf[d] = __builtin_amdgcn_raw_buffer_load_b128(xrs, c < c_hi ? xo + at : VO_OUTSIDE, 0, 0);
            } else {
                wf[d] = vo_load_unaligned<T>(w + (int64_t)fr * a.C + c, fr < rows_w ? c_hi - c : 0, c);
                xf[d] = vo_load_unaligned<T>(x + fr * a.xs + c, fr < a.M ? c_hi - c : 0, c);
            }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
#pragma unroll
            for (int part = 0; part < vo_elem<T>::PARTS; ++part) acc = vo_elem<T>::mma16(wf[d], xf[d], acc, part);
    }
    *reinterpret_cast<vo_f32x4*>(&sums[wave][fr][fg * 4]) = acc;
    __syncthreads();
    constexpr int ACROSS = 16 / PER;
    const int r = threadIdx.x / ACROSS, k = threadIdx.x % ACROSS * PER;
    if (r >= 16 || r >= a.M || n0 + k >= a.K) return;
    Piece<T> p;
    float v[PER] = {}, bias[PER];
    p.load_residual(a, r, n0 + k);
    Piece<T>::load_bias(a, n0 + k, bias);
#pragma unroll
    for (int s = 0; s < NW; ++s)
#pragma unroll
        for (int q = 0; q < PER; ++q) v[q] += sums[s][r][k + q];
    p.emit(a, split, r, n0 + k, v, bias);
}

// Adds the partial sums of one PER-wide piece in the order of the splits and finishes it.
template <typename T> __global__ __launch_bounds__(256) void linear_join(const LinArgs a) {
    constexpr int PER = vo_elem<T>::PER;
    const int64_t across = (a.K + PER - 1) / PER, piece = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (piece >= a.M * across) return;
    const int64_t m = piece / across;
    const int k = (int)(piece % across) * PER;
    Piece<T> piece_of;
    float v[PER] = {}, bias[PER];
    piece_of.load_residual(a, m, k);
    Piece<T>::load_bias(a, k, bias);
    const bool wide = k + PER <= a.K;
    for (int s = 0; s < a.splits; ++s) {
        const float* p = a.part + ((int64_t)s * a.M + m) * a.K + k;
        if (wide) {
#pragma unroll
            for (int j = 0; j < PER; j += 4) {
                const vo_f32x4 t = __builtin_bit_cast(vo_f32x4, vo_load16(p + j));
                v[j] += t[0]; v[j + 1] += t[1]; v[j + 2] += t[2]; v[j + 3] += t[3];
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] += k + j < a.K ? p[j] : 0.f;
        }
    }
    piece_of.finish(a, m, k, v, bias);
}

// Rows of C elements, any alignment, to rows of C rounded up to whole 16-byte pieces: x behind one another, then W.
template <typename T> __global__ __launch_bounds__(256) void linear_pad(const T* x, int64_t xs, int64_t M, const T* w, int K, int C, T* out) {
    constexpr int PER = vo_elem<T>::PER;
    const int64_t across = (C + PER - 1) / PER, piece = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (piece >= (M + K) * across) return;
    const int64_t row = piece / across;
    const int c = (int)(piece % across) * PER;
    const T* p = row < M ? x + row * xs : w + (row - M) * C;
    *reinterpret_cast<vo_u32x4*>(out + piece * PER) = vo_load_unaligned<T>(p + c, C - c, c);
}

// ------------------------------------------------------------------------------------------------------------- host

// Tiles: rows of x, outputs; the share of the CU's rate that a tile reaches on a long C, in 16 bits and in float32; the C at which
// half of that is reached (an eighth of it in float32, whose products take longer).
// Measured on 16-bit products, us: 4096 x 4096 x 4096 on forms 3 / 4: 152 / 123; 2048 x 2048 x 2048 on 2 / 3 / 4: 32 / 36 / 49;
// 38400 x 256 x 256 on 2 / 3 / 4: 19 / 25 / 26; float32: 38400 x 256 x 256 on 2 / 3: 63 / 72, 4096 x 4096 x 4096: 985 / 973.
struct Form { int bm, bn; float rate16, rate32, ramp; };
constexpr Form FORMS[] = {{16, 16, 0, 0, 0}, {32, 64, 0, 0, 0}, {64, 64, 0.55f, 1.f, 100}, {128, 128, 0.75f, 1.05f, 500}, {256, 256, 1.f, 0.f, 800}};

struct Plan {
    int form;                        // of FORMS; 0: linear_rows
    int splits, c_per_split;
    int64_t tiles_m, tiles_n;
    bool deep;                       // few 64 x 64 tiles: more slabs under way in place of more workgroups
    int64_t padded;                  // C not in whole 16-byte pieces: elements of the padded copies of x and W (0: none are made)
};

Plan plan(int64_t M, int C, int K, int dtype) {
    const int slab = dtype == VO_F32 ? 32 : 64, per = slab / 8;
    Plan p{};
    // Unaligned rows cannot go straight into LDS, and through registers they run at less than half the rate: where the product
    // outweighs its operands they are copied to aligned rows first (3001 x 2777 x 3333 bfloat16: 183 us without the copies).
    if (C % per && (double)M * K >= (dtype == VO_F32 ? 96. : 512.) * (M + K) && (double)M * K * C >= 1e9) {
        C = (C + per - 1) / per * per;
        p.padded = (M + K) * C;
    }
    if (M <= 32) {
        // One row of 4096 x 4096 (bfloat16): 10 us by rows, 12 by split tiles and their join; 16 rows of 4096 x 16384: 39 by
        // rows, 31 by tiles that need no split.
        p.form = M <= 4 || (M <= 16 && vo_ceil_div(K, 64) < 192) ? 0 : 1;
    }
    int64_t splits = 1;
    if (M <= 32) {
        const int64_t tiles = vo_ceil_div(M, FORMS[p.form].bm) * vo_ceil_div(K, FORMS[p.form].bn);
        // elements of C worth a part (19 rows of 2533 float32 by 1434: 25 us in 4 parts, 19 in 8; one of 1800 by 226: 6 unsplit, 7 in 2)
        const int64_t at_least = p.form == 0 ? 1024 : dtype == VO_F32 ? 256 : 512;
        if (tiles < 192) splits = vo_ceil_div(256, tiles);
        if (splits > C / at_least) splits = C / at_least;
        if (splits > 16) splits = 16;
        if (splits < 1) splits = 1;
    } else {
        // The form and the number of parts of C whose estimated time is least: rounds over the 256 CUs times a part's time, and
        // the join's launch and traffic.  Fewer workgroups than two per CU do not hide their waits.
        double best = 0.;
        for (int f = 2; f <= 4; ++f) {
            const Form& form = FORMS[f];
            const double rate = dtype == VO_F32 ? form.rate32 * 0.5e6 : form.rate16 * 4.7e6;        // operations per CU and us
            if (rate == 0.) continue;
            const double ramp = dtype == VO_F32 ? form.ramp / 8 : form.ramp;
            const int64_t tiles = vo_ceil_div(M, form.bm) * vo_ceil_div(K, form.bn);
            for (int n = 1; n <= 16 && (n == 1 || C / n >= 256); ++n) {
                const int64_t blocks = tiles * n, rounds = vo_ceil_div(blocks, 256);
                const double full = f == 4 ? 1. : blocks <= 256 ? 0.6 : blocks <= 512 ? 0.85 : 1.;
                const double us = rounds * 2. * form.bm * form.bn * ((double)C / n + ramp) / (rate * full) +
                                  (n > 1 ? 4. + n * (double)M * K * 8 / 4e6 : 0.);
                if (p.form == 0 || us < best) {
                    best = us;
                    p.form = f;
                    splits = n;
                }
            }
        }
    }
    p.tiles_m = vo_ceil_div(M, FORMS[p.form].bm);
    p.tiles_n = vo_ceil_div(K, FORMS[p.form].bn);
    const int64_t tiles = p.tiles_m * p.tiles_n;
    p.c_per_split = (int)vo_ceil_div(vo_ceil_div(C, slab), splits) * slab;
    p.splits = (int)vo_ceil_div(C, p.c_per_split);
    p.deep = tiles * p.splits <= 512;                                // 512 x 2048 x 2048: 14 us against 20; 2048^3: 37 against 32
    return p;
}

// A launch has fewer than 2^32 threads.  Sizes that pass this by far (2^23 tiles of the largest size) are told first: the products in
// plan() could pass 64 bits.
bool too_large(int64_t M, int K) { return (double)M * K >= (double)(1ll << 39); }

int64_t needed(const Plan& p, int64_t M, int K, int dtype) {
    return p.padded * (dtype == VO_F32 ? 4 : 2) + (p.splits > 1 ? (int64_t)p.splits * M * K * 4 : 0);
}

template <typename T, bool DIRECT> int launch(const LinArgs& a, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n * p.splits));
    constexpr int S32 = DIRECT ? 6 : 2, S64 = DIRECT ? 4 : 2;        // slabs under way
    if (p.form == 0) linear_rows<T, DIRECT><<<grid, 512, 0, st>>>(a);
    else if (p.form == 1) linear_tiles<T, 32, 64, 1, 4, S32, DIRECT><<<grid, 256, 0, st>>>(a);
    else if (p.form == 2 && p.deep) linear_tiles<T, 64, 64, 2, 2, S64, DIRECT><<<grid, 256, 0, st>>>(a);
    else if (p.form == 2) linear_tiles<T, 64, 64, 2, 2, 2, DIRECT><<<grid, 256, 0, st>>>(a);
    else if (p.form == 3) linear_tiles<T, 128, 128, 2, 2, 2, DIRECT><<<grid, 256, 0, st>>>(a);
    else if constexpr (sizeof(T) == 2 && DIRECT) linear_tiles<T, 256, 256, 2, 4, 2, DIRECT><<<grid, 512, 0, st>>>(a);
    VO_CHECK_LAUNCH("vo_linear");
    if (p.splits > 1) {
        const int64_t pieces = a.M * vo_ceil_div(a.K, vo_elem<T>::PER);
        linear_join<T><<<dim3((unsigned)vo_ceil_div(pieces, 256)), 256, 0, st>>>(a);
        VO_CHECK_LAUNCH("vo_linear (join)");
    }
    return VO_OK;
}

template <typename T> int dispatch(LinArgs a, Plan p, hipStream_t st) {
    const size_t es = sizeof(T);
    if (p.padded) {
        T* rows = reinterpret_cast<T*>(a.part);
        linear_pad<T><<<dim3((unsigned)vo_ceil_div(p.padded / vo_elem<T>::PER, 256)), 256, 0, st>>>(
            static_cast<const T*>(a.x), a.xs, a.M, static_cast<const T*>(a.w), a.K, a.C, rows);
        VO_CHECK_LAUNCH("vo_linear (padded rows)");
        a.C = (int)(p.padded / (a.M + a.K));
        a.x = rows;
        a.xs = a.C;
        a.w = rows + a.M * a.C;
        a.part = reinterpret_cast<float*>(rows + p.padded);
    }
    const bool direct = (a.C * es) % 16 == 0 && (a.xs * es) % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
    if (!direct && p.form == 4) {                                    // registers for staging leave no room for the largest tile
        p.form = 3;
        a.tiles_m = (unsigned)(p.tiles_m = vo_ceil_div(a.M, 128));
        a.tiles_n = (unsigned)(p.tiles_n = vo_ceil_div(a.K, 128));
    }
    return direct ? launch<T, true>(a, p, st) : launch<T, false>(a, p, st);
}

}  // namespace

extern "C" int64_t vo_linear_workspace_bytes(int64_t M, int C, int K, int dtype) {
    if (M <= 0 || C <= 0 || K <= 0 || too_large(M, K)) return 0;
    return needed(plan(M, C, K, dtype), M, K, dtype);
}

extern "C" int vo_linear(const void* x, int64_t x_row_stride, const void* weight, const float* bias, const void* residual,
                         int64_t residual_row_stride, void* y, int64_t y_row_stride, int64_t M, int C, int K, int activation,
                         int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    VO_REQUIRE(dtype == VO_F32 || dtype == VO_F16 || dtype == VO_BF16, "vo_linear: dtype=%d is none of VO_F32, VO_F16, VO_BF16", dtype);
    VO_REQUIRE(activation >= VO_ACT_NONE && activation <= VO_ACT_SILU, "vo_linear: unknown activation %d", activation);
    VO_REQUIRE(M >= 0 && C >= 1 && K >= 1, "vo_linear: M=%lld C=%d K=%d (M >= 0, C >= 1, K >= 1 required)", (long long)M, C, K);
    if (M == 0) return VO_OK;
    VO_REQUIRE(x && weight && y, "vo_linear: null pointer");
    VO_REQUIRE(x_row_stride >= C && y_row_stride >= K && (!residual || residual_row_stride >= K || residual_row_stride == 0),
               "vo_linear: row strides must be at least the rows' lengths (the residual's may be 0)");
    const int64_t es = dtype == VO_F32 ? 4 : 2;
    // a tile's rows are addressed with 32-bit offsets
    if (x_row_stride * es * 256 >= (1ll << 31) || (int64_t)C * es * 256 >= (1ll << 31))
        return vo_fail(VO_ERR_UNSUPPORTED, "vo_linear: rows of x and weight must be under 8 MiB");
    const bool large = too_large(M, K);
    const Plan p = large ? Plan{} : plan(M, C, K, dtype);
    const int64_t limit = 1ll << 32;                                 // (large forms may be run as tiles of half the side)
    if (large || p.tiles_m * p.tiles_n * p.splits * (p.form == 0 ? 512 : 1024) >= limit || M * vo_ceil_div(K, 4) >= limit * 64 ||
        (p.splits > 1 && M * vo_ceil_div(K, 16 / es) >= limit) || p.padded / (16 / es) >= limit)
        return vo_fail(VO_ERR_UNSUPPORTED, "vo_linear: M=%lld C=%d K=%d is too large for one launch", (long long)M, C, K);
    const int64_t need = needed(p, M, K, dtype);
    VO_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               "vo_linear: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    LinArgs a{};
    a.x = x; a.w = weight; a.bias = bias; a.res = residual; a.y = y; a.part = static_cast<float*>(workspace);
    a.xs = x_row_stride; a.rs = residual_row_stride; a.ys = y_row_stride;
    a.M = M; a.C = C; a.K = K; a.act = activation;
    a.splits = p.splits; a.c_per_split = p.c_per_split;
    a.tiles_m = (unsigned)p.tiles_m; a.tiles_n = (unsigned)p.tiles_n;
    hipStream_t st = vo_stream(stream);
    if (dtype == VO_F32) return dispatch<float>(a, p, st);
    if (dtype == VO_F16) return dispatch<_Float16>(a, p, st);
    return dispatch<__bf16>(a, p, st);
}
