// Attention of packed sequences: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys a row sees.
//   q, out (Tq,Hq,D), k, v (Tk,Hk,D) in float32, float16 or bfloat16; head h reads key head h / (Hq/Hk); sequence s owns
//   the rows [q_offsets[s], q_offsets[s+1]) and the keys [k_offsets[s], k_offsets[s+1]); causal: row i of Lq sees the
//   keys j <= i + Lk - Lq.  A row that sees nothing gives 0.
//
// One pass over the keys with a running maximum m and sum l per row.  Both products run on the matrix cores, transposed:
//   S^T = K Q^T   lane l holds column q = l % 32 and the keys 8 b + 4 (l / 32) + i of a block of 32 (b, i = 0..3)
//   O^T = V^T P^T wants column q = l % 32 and, from lane half l / 32, half of the keys of each step: whichever half of the
//                 keys that is, the sum over keys is the same as long as V^T is read in the same order.  So the exponentials
//                 are already where the second product needs them: they are rounded to the 16-bit type in place (float32: not
//                 at all) and no value crosses lanes.  m, l and the rescaling factor are one number per lane.
// The rounding is what the 16-bit product takes; it carries the result's error from its own rounding's 0.0017 (bfloat16, relative to
// 64 bits) to 0.0022, in float16 from 0.00021 to 0.00029.  To multiply the remainder too would be half as many products again.
// V^T in 16 bits comes out of LDS by the transposing read: four keys of one feature per lane.
//
// The exponent's argument is (s - m) * scale * log2(e), with the difference formed first: s c - m c in one fused multiply-add would
// leave the rounding of m c in it, which is 16 and more where scores times c pass 2^28 (no weight would be near 1, sums would vanish or
// overflow).  The instruction more costs the prompts below 1.5 %, heads of 32 features 8 %; both forms under a test of |m c| spill.
// m follows the true maximum only when it has grown by more than 2^8 in the exponentials, so most tiles need no
// rescaling of the sums (the exponentials are then at most 256, which costs no bits in a floating-point format).  In float16 they are
// kept 2^7 up, sums included: its smallest number is 2^-24, and thousands of keys below that beside one large one weigh something together.
//
// Two forms:
//   tiles  a workgroup of four waves takes 128 rows of one key head (a row is a token and one of the heads that share the key
//          head); key tiles are shared in LDS, loaded while the previous tile is multiplied.  Matrix and vector work of a tile
//          take about as long as each other and overlap between the two to four workgroups of a CU; the chip's power sets the
//          clock (the same cycles are 38 % faster on zeros).  8 prompts of up to 8192 tokens, 32 / 8 heads of 128, bfloat16,
//          causal: 2.09 ms = 1.00 PFLOP/s; 4800 float32 rows, 4 heads of 64: 204 us = 116 TFLOP/s of the 153 the library's
//          product reaches.
//   rows   few rows per sequence (single tokens above all): tiles of 32 rows, every wave streams key tiles of its own into its
//          own part of LDS, the waves' results are joined at the end.  Bound by the read of keys and values: 32 caches of up to
//          32768 tokens, 8 key heads of 128: 363 us = 5.4 TB/s; a single row before 777 keys 12 us, all of it waiting.
// Either can be split over the keys; the parts (m, l, unnormalised sums) go to a workspace and are joined in a fixed order.
#include "vo_packed.h"
#include "vo_tokens.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;

struct AttArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* part;                                  // splits > 1: sums (splits, Tq, Hq, D), then m and l (splits, Tq, Hq, 2)
    const int* q_off;
    const int* k_off;
    int64_t qs, qh, ks, kh, vs, vh, os, oh;       // token and head strides in elements
    int64_t Tq, Tk;
    int sequences, Hq, Hk, group, D, causal, splits;
    unsigned tiles;                               // row tiles over all sequences (an upper bound)
    unsigned reciprocal;                          // 2^16 / group rounded up, 0 for groups over 128
    float c;                                      // scale * log2(e)
};

// Key tiles in LDS: rows of DT elements in 16-byte chunks, permuted within each row.  K is read 16 rows of one chunk at a time,
// V (16 bits) four rows of 64 bytes, V (float32) two rows of 128 bytes four rows apart: each permutation spreads its reader's
// bytes over all 64 banks.  It is an exclusive or where the number of chunks is a power of two, else (DT = 96: two rows
// in four, or one in two, start at another bank already) a rotation.
template <typename T, int DT> struct Tile {
    static constexpr int ES = sizeof(T), PER = vo_elem<T>::PER, CH = DT / PER, ROW = DT * ES;
    static constexpr bool POW2 = (CH & (CH - 1)) == 0;
    static constexpr int PER_LINE = ROW >= 256 ? 1 : 256 / ROW;      // rows in 256 bytes
    static constexpr int KMASK = CH < 16 ? CH - 1 : 15;
    static __device__ __forceinline__ int k_swz(int r) { return POW2 ? (r / PER_LINE) & KMASK : (r & 31) >> (ES == 4 ? 1 : 2); }
    static __device__ __forceinline__ int v_swz(int r) {
        if constexpr (ES == 4) return CH > 8 ? ((r >> 2) & 1) << 3 : 0;
        return !POW2 || CH <= 4 ? 0 : CH == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
    }
    static __device__ __forceinline__ int place(int chunk, int swz) {        // where a chunk lies
        if constexpr (POW2) return chunk ^ swz;
        return chunk + swz < CH ? chunk + swz : chunk + swz - CH;
    }
    static __device__ __forceinline__ int chunk_at(int place, int swz) {     // which chunk lies there
        if constexpr (POW2) return place ^ swz;
        return place < swz ? place + CH - swz : place - swz;
    }
};

// 32 rows of one wave against key tiles.
template <typename T, int DT, int KEYS> struct Core {
    using E = vo_elem<T>;
    using L = Tile<T, DT>;
    static constexpr int QS = DT / (2 * E::PER), KB = KEYS / 32, DB = DT / 32;
    vo_u32x4 q[QS];
    vo_f32x16 o[DB];
    float m, l;                                   // m: the maximum of the scores s = q.k (not scaled) that the sums refer to

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }
    // p: this lane's row (null: no row), chunks of D elements
    __device__ __forceinline__ void load_q(const T* p, int D, int lane) {
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const int c = s * 2 + (lane >> 5);
            q[s] = p && c * E::PER < D ? *reinterpret_cast<const vo_u32x4*>(p + c * E::PER) : vo_u32x4{0, 0, 0, 0};
        }
    }
    // s = K q of a key tile
    __device__ __forceinline__ void scores(const unsigned char* kt, vo_f32x16* s, int lane) const {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            vo_u32x4 k[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int r = b * 32 + (lane & 31);
                k[b] = *reinterpret_cast<const vo_u32x4*>(kt + r * L::ROW + L::place(i * 2 + (lane >> 5), L::k_swz(r)) * 16);
            }
#pragma unroll
            for (int part = 0; part < E::PARTS; ++part)
#pragma unroll
                for (int b = 0; b < KB; ++b) s[b] = E::mma32(k[b], q[i], s[b], part);
        }
    }
    // The lane's row sees the tile's keys below `limit`.
    static __device__ __forceinline__ void mask(vo_f32x16* s, int limit, int lane) {
        const int mine = limit - 4 * (lane >> 5);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (b * 32 + 8 * (i >> 2) + (i & 3) >= mine) s[b][i] = -INFINITY;
    }
    // The largest of this lane's scores.
    static __device__ __forceinline__ float largest(const vo_f32x16* s) {
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        return top;
    }
    // Lets m follow the row's largest score (`top`: this half's) where that pays (see the top of the file).
    __device__ __forceinline__ void follow(float top, float c) {
        top = across(top, [](float x, float y) { return fmaxf(x, y); });
        if (__any((top - m) * c > 8.f)) {                            // m starts at -inf; -inf - -inf is no reason either
            const float next = fmaxf(m, top);
            const float f = next == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
            l *= f;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= f;
            m = next;
        }
    }
    static __device__ __forceinline__ float weight(float s, float c, float ref) {
        return __builtin_amdgcn_exp2f(__is_same(T, _Float16) ? __builtin_fmaf(s - ref, c, 7.f) : (s - ref) * c);
    }
    // Scores 2 j and 2 j + 1 of a block of 32 keys to exponentials, rounded to the storage type where that has 16 bits; `sum` takes
    // the unrounded ones.
    static constexpr int PW = sizeof(T) == 2 ? 8 : 16;               // registers of a block's exponentials
    static __device__ __forceinline__ void weigh(const vo_f32x16& s, unsigned* p, float* sum, int j, float c, float ref) {
        const float x = weight(s[2 * j], c, ref), y = weight(s[2 * j + 1], c, ref);
        sum[0] += x;
        sum[1] += y;
        if constexpr (sizeof(T) == 2) {
            p[j] = E::pack2(x, y);
        } else {
            p[2 * j] = __builtin_bit_cast(unsigned, x);
            p[2 * j + 1] = __builtin_bit_cast(unsigned, y);
        }
    }
    __device__ __forceinline__ void weights(const vo_f32x16* s, unsigned (*p)[PW], float c) {
        const float ref = m == -INFINITY ? 0.f : m;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8 * KB; ++j) weigh(s[j / 8], p[j / 8], sum, j % 8, c, ref);
        l += sum[0] + sum[1];
    }
    // 16 bits: V^T of 16 keys (half `h` of block b) for every 32 features.  Keys r.. and r + 8.. : the lane supplies 8 bytes of row
    // r + (lane % 16) / 4 and receives four rows of feature d * 32 + lane % 32.
    // One piece is 16 keys of one block of features, the operand of one product: piece j has the features j % DB, the keys 16 (j / DB)...
    static constexpr int VALUES = 2 * KB * DB;
    static __device__ __forceinline__ vo_u32x4 value_piece(const unsigned char* vt, int j, int lane) {
        const int r = 16 * (j / DB) + 4 * (lane >> 5) + ((lane & 15) >> 2), at = (lane & 1) * 8;
        const int chunk = j % DB * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const vo_u32x2 lo = transposed(vt + r * L::ROW + L::place(chunk, L::v_swz(r)) * 16 + at);
        const vo_u32x2 hi = transposed(vt + (r + 8) * L::ROW + L::place(chunk, L::v_swz(r + 8)) * 16 + at);
        return vo_u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    __device__ __forceinline__ void add_values(vo_u32x4 v, const unsigned (*p)[PW], int j) {
        const unsigned* w = p[j / (2 * DB)] + 4 * (j / DB % 2);
        o[j % DB] = E::mma32(v, vo_u32x4{w[0], w[1], w[2], w[3]}, o[j % DB], 0);
    }
    // o += V^T p
    __device__ __forceinline__ void accumulate(const unsigned char* vt, const unsigned (*p)[PW], int lane) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < VALUES; ++j) add_values(value_piece(vt, j, lane), p, j);
            return;
        }
        const int col = lane & 31, half = lane >> 5;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = b * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const int chunk = d * 8 + (col >> 2);
                    const float vf = *reinterpret_cast<const float*>(vt + r * L::ROW + L::place(chunk, L::v_swz(r)) * 16 + (col & 3) * 4);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, __builtin_bit_cast(float, p[b][i]), o[d], 0, 0, 0);
                }
            }
    }
    // Values that are infinite or NaN ("unbounded").  Where all rows see the same keys they are products like others; where a row
    // does not see a key its weight is zero, and zero times such a value is no zero.  So a tile on a causal sequence's diagonal (or
    // at the end of tokens that overlap in memory) that holds any is multiplied with zeros in their place, and their products are
    // added at the end to the rows that see them: the value itself (any positive weight times it is it), or NaN where the weight
    // beside the row's largest is zero all the same.
    static constexpr unsigned EXP = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    static __device__ __forceinline__ bool unbounded(unsigned bits) { return (bits & EXP) == EXP; }
    // Is there any in the tile?
    static __device__ __forceinline__ bool any_unbounded(const unsigned char* vt, int lane) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        unsigned top[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KEYS * L::ROW / 1024; ++i) {
            const vo_u32x4 x = *reinterpret_cast<const vo_u32x4*>(vt + i * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 2)
                    top[j] = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top[j]), __builtin_bit_cast(u16x2, x[j] & 0x7fff7fffu)));
                else
                    top[j] = max(top[j], x[j] & 0x7fffffffu);
            }
        }
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= unbounded(top[j]) || (sizeof(T) == 2 && unbounded(top[j] >> 16));
        return __any(bad);
    }
    static __device__ __forceinline__ unsigned bounded(unsigned x) {
        if constexpr (sizeof(T) == 4) return unbounded(x) ? 0u : x;
        return (unbounded(x) ? 0u : x & 0xffffu) | (unbounded(x >> 16) ? 0u : x & 0xffff0000u);
    }
    // Part `share` of `shares` of the tile's values: unbounded ones become zero.
    static __device__ __forceinline__ void bound(unsigned char* vt, int share, int shares, int lane) {
#pragma unroll 1
        for (int i = share; i < KEYS * L::ROW / 1024; i += shares) {
            vo_u32x4* x = reinterpret_cast<vo_u32x4*>(vt + i * 1024 + lane * 16);
            *x = vo_u32x4{bounded((*x)[0]), bounded((*x)[1]), bounded((*x)[2]), bounded((*x)[3])};
        }
    }
    // The products of the unbounded values of the tile's `keys` keys, in memory from `v` on, added to the sums; kt: the keys.  The scores
    // are formed once more: to keep the weights' zeros from the loop would cost its kernels registers that they spill.
    __device__ __forceinline__ void add_unbounded(const unsigned char* kt, const T* v, int64_t stride, int keys, int limit, float c, int D, int lane) {
        vo_f32x16 s[KB];
        unsigned none[KB];                                           // the row's keys of weight zero: a bit for each of a block's 32
        scores(kt, s, lane);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            unsigned u = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = weight(s[b][i], c, ref);
                bool zero = w == 0.f;
                if constexpr (sizeof(T) == 2) zero = (E::pack2(w, 0.f) & 0x7fffu) == 0;
                u |= (unsigned)zero << (8 * (i >> 2) + (i & 3));
            }
            const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            none[b] = both[0] | both[1] << 4;                        // the upper half of the wave holds the keys four further
        }
#pragma unroll 1
        for (int r = 0; r < keys; ++r) {
            unsigned u = none[0];
#pragma unroll
            for (int b = 1; b < KB; ++b) u = r >> 5 == b ? none[b] : u;
            const bool zero = u >> (r & 31) & 1;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int f = d * 32 + 8 * b + 4 * (lane >> 5);
                    if (f >= D || r >= limit) continue;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x = E::get(v + r * stride + f + j);
                        if (!(fabsf(x) < INFINITY)) o[d][4 * b + j] += zero ? NAN : x;
                    }
                }
        }
    }
    // A whole tile.
    __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, float c, bool masked, int limit, int lane) {
        vo_f32x16 s[KB];
        unsigned p[KB][PW];
        scores(kt, s, lane);
        if (masked) mask(s, limit, lane);
        follow(largest(s), c);
        weights(s, p, c);
        accumulate(vt, p, lane);
    }
    // x of this lane and of the other half's lane (l + 32) % 64, combined: both get the same
    template <typename F> static __device__ __forceinline__ float across(float x, F f) {
        const unsigned u = __builtin_bit_cast(unsigned, x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned lo = r[0], hi = r[1];
        return f(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
    }
    static __device__ __forceinline__ vo_u32x2 transposed(const unsigned char* p) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(vo_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
    }
};

// A wave's share of the 16-byte pieces of one operand's key tile: N loads of 64 pieces.
template <typename T, int DT, int KEYS, int WAVES> struct Loader {
    using L = Tile<T, DT>;
    static constexpr int N = KEYS * L::CH / 64 / WAVES;
    static_assert(N >= 1 && KEYS * L::CH % (64 * WAVES) == 0, "a key tile must be whole wave loads");
    unsigned off[N];
    __device__ __forceinline__ void init(int64_t stride, int D, bool is_v, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int piece = (wave * N + i) * 64 + lane, r = piece / L::CH;
            const int chunk = L::chunk_at(piece % L::CH, is_v ? L::v_swz(r) : L::k_swz(r));
            off[i] = chunk * L::PER < D ? (unsigned)(r * stride * L::ES) + chunk * 16 : VO_OUTSIDE;
        }
    }
    // base: the tile's first key; keys: how many there are (the rest of the tile becomes zero)
    __device__ __forceinline__ void load(const T* base, int64_t stride, int64_t keys, int D, unsigned char* lds, int wave) const {
        const int64_t n = keys < KEYS ? keys : KEYS;
        const __amdgpu_buffer_rsrc_t rs = vo_buffer(base, n > 0 ? ((n - 1) * stride + D) * L::ES : 0);
#pragma unroll
        for (int i = 0; i < N; ++i) vo_load_to_lds(rs, lds + (wave * N + i) * 1024, off[i]);
    }
};

// A result in 16 bits.  The weights of the sum are rounded, the sum of weights that divides it is not: a mean of numbers near the
// type's largest may pass it by a rounding, but is finite like them.
template <typename T> constexpr float LARGEST = __is_same(T, _Float16) ? 65504.f : __is_same(T, __bf16) ? 0x1.fep127f : INFINITY;
template <typename T> __device__ __forceinline__ float in_range(float x) {
    if constexpr (sizeof(T) == 4) return x;
    return fabsf(x) < INFINITY ? fminf(fmaxf(x, -LARGEST<T>), LARGEST<T>) : x;
}

// Where the results of a row go: the output, or (split) the workspace.
__device__ __forceinline__ float* part_row(const AttArgs& a, int split, int64_t token, int head) {
    return a.part + (((int64_t)split * a.Tq + token) * a.Hq + head) * a.D;
}
__device__ __forceinline__ float* part_ml(const AttArgs& a, int split, int64_t token, int head) {
    return a.part + (int64_t)a.splits * a.Tq * a.Hq * a.D + (((int64_t)split * a.Tq + token) * a.Hq + head) * 2;
}
template <typename T> __device__ __forceinline__ T* out_row(const AttArgs& a, int64_t token, int head) {
    return static_cast<T*>(a.out) + token * a.os + head * a.oh;
}

// A wave's O^T (times `factor`, one number per lane = row) as rows of S: a lane holds four features of one row at a time, so
// the rows are put together in the wave's own LDS (chunks in an order that spreads the banks) and leave in pieces of 16 bytes.
// row(r): where row r goes, null if it does not exist.
template <typename S, int DT, typename F>
__device__ __forceinline__ void store_rows(const vo_f32x16* o, float factor, int D, unsigned char* lds, int lane, F row) {
    using L = Tile<S, DT>;
    constexpr int ES = sizeof(S), CH = L::CH, EACH = L::PER;
    auto swz = [](int r) { return L::POW2 ? r & L::KMASK : L::k_swz(r); };
    const int r = lane & 31;
    auto put = [&](auto result) {
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int f = d * 32 + 8 * b + 4 * (lane >> 5);
                unsigned char* p = lds + r * DT * ES + L::place(f / EACH, swz(r)) * 16 + f % EACH * ES;
                const float v0 = result(o[d][4 * b]), v1 = result(o[d][4 * b + 1]), v2 = result(o[d][4 * b + 2]), v3 = result(o[d][4 * b + 3]);
                if constexpr (ES == 2) *reinterpret_cast<vo_u32x2*>(p) = vo_u32x2{vo_elem<S>::pack2(v0, v1), vo_elem<S>::pack2(v2, v3)};
                else *reinterpret_cast<vo_f32x4*>(p) = vo_f32x4{v0, v1, v2, v3};
            }
    };
    float top = 0.f;                                                 // of the numbers: one test for all of a lane's
    if constexpr (ES == 2) {
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(o[d][i]));
    }
    if (ES == 2 && __any(top * factor > LARGEST<S>)) put([&](float x) { return in_range<S>(x * factor); });
    else put([&](float x) { return x * factor; });
    vo_wave_lds_fence();
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        const int piece = i * 64 + lane, q = piece / CH, c = L::chunk_at(piece % CH, swz(q));
        S* p = row(q);
        if (p && c * EACH < D) *reinterpret_cast<vo_u32x4*>(p + c * EACH) = *reinterpret_cast<const vo_u32x4*>(lds + piece * 16);
    }
}

__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }      // 0: the row saw nothing

// ------------------------------------------------------------------------------------------------------------ tiles
template <typename T, int DT, int KEYS, int MIN_BLOCKS>
__global__ __launch_bounds__(256, MIN_BLOCKS) void attention_tiles(const AttArgs a) {
    using L = Tile<T, DT>;
    constexpr int ROWS = 128, HALF = KEYS * L::ROW;
    static_assert(HALF >= 32 * DT * 4, "a wave's rows of float32 fit a quarter of the LDS");
    __shared__ __align__(16) unsigned char lds[4 * HALF];            // two stages of K and V
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // numbers: key head outermost (an XCD keeps to few of them: their keys stay in its L2), then split, then row tiles from
    // the last (the longest ones of a causal sequence come first)
    const unsigned id = vo_xcd_contiguous(blockIdx.x, gridDim.x);
    const unsigned tile = a.tiles - 1 - id % a.tiles;
    const int split = id / a.tiles % a.splits, kh = id / a.tiles / a.splits;
    const vo_place p = vo_find_tile(a.q_off, a.k_off, a.sequences, a.Tq, a.Tk, tile, a.group, ROWS);
    if (!p.any) return;

    // row r of the tile is head (r + skew) % group of token (r + skew) / group, counted from the tile's first token
    const int64_t shift = p.Lk - p.Lq, first_token = p.row / a.group;
    const int skew = (int)(p.row - first_token * a.group);
    const int rows = (int)(p.Lq * a.group - p.row < ROWS ? p.Lq * a.group - p.row : ROWS);
    // (x / group by multiplication: exact while x times the reciprocal's excess, under 256 * 128, stays below 2^16)
    auto by_group = [&](unsigned x) { return a.reciprocal ? x * a.reciprocal >> 16 : x / (unsigned)a.group; };
    auto token_of = [&](int r) { return first_token + by_group(r + skew); };
    auto head_of = [&](int r) { return kh * a.group + (int)(r + skew - by_group(r + skew) * a.group); };
    int64_t seen = a.causal ? token_of(rows - 1) + 1 + shift : p.Lk;                         // keys that some row sees
    seen = vo_clamp64(seen, 0, p.Lk);
    const int64_t key_tiles = (seen + KEYS - 1) / KEYS, per = (key_tiles + a.splits - 1) / a.splits;
    const int64_t t0 = split * per < key_tiles ? split * per : key_tiles, t1 = t0 + per < key_tiles ? t0 + per : key_tiles;

    const int first = wave * 32, row = first + (lane & 31);
    const bool have = row < rows;
    const int64_t token = token_of(row);
    const int head = head_of(row);
    Core<T, DT, KEYS> core;
    core.reset();
    core.load_q(have ? static_cast<const T*>(a.q) + (p.q0 + token) * a.qs + head * a.qh : nullptr, a.D, lane);
    // keys below `limit` are seen by this lane's row; tiles wholly below wave_all need no mask, from wave_any on no work; tiles
    // wholly below `all` are seen by every row of the workgroup
    const int64_t limit = a.causal ? vo_clamp64(token + shift + 1, 0, p.Lk) : p.Lk;
    int64_t all = a.causal ? vo_clamp64(first_token + shift + 1, 0, p.Lk) : p.Lk;
    if (a.vs < a.D && all == p.Lk) --all;                            // tokens overlap: a tile at their end holds parts of tokens behind the last
    int64_t unbounded = t1;                                          // the first tile that was bounded
    const int64_t wave_all = a.causal ? vo_clamp64(token_of(first) + shift + 1, 0, p.Lk) : p.Lk;
    const int64_t wave_any = first >= rows ? 0 : a.causal ? vo_clamp64(token_of(first + 31) + shift + 1, 0, p.Lk) : p.Lk;

    const T* kb = static_cast<const T*>(a.k) + p.k0 * a.ks + kh * a.kh;
    const T* vb = static_cast<const T*>(a.v) + p.k0 * a.vs + kh * a.vh;
    Loader<T, DT, KEYS, 4> lk, lv;
    lk.init(a.ks, a.D, false, wave, lane);
    lv.init(a.vs, a.D, true, wave, lane);
    auto fetch_k = [&](int64_t t, unsigned char* buf) { lk.load(kb + t * KEYS * a.ks, a.ks, p.Lk - t * KEYS, a.D, buf, wave); };
    auto fetch_v = [&](int64_t t, unsigned char* buf) { lv.load(vb + t * KEYS * a.vs, a.vs, p.Lk - t * KEYS, a.D, buf, wave); };
    unsigned char *now = lds, *next = lds + 2 * HALF;
    if (t0 < t1) {
        fetch_k(t0, now);
        fetch_v(t0, now + HALF);
    }
    for (int64_t t = t0; t < t1; ++t) {
        vo_lds_barrier();                                        // tile t has arrived, tile t - 1 has been read
        if (t + 1 < t1) {
            fetch_k(t + 1, next);
            fetch_v(t + 1, next + HALF);
        }
        const int64_t key = t * KEYS;
        if (key + KEYS > all && all < p.Lk && core.any_unbounded(now + HALF, lane)) {        // all waves find the same
            vo_lds_barrier();
            core.bound(now + HALF, wave, 4, lane);
            vo_lds_barrier();
            unbounded = t < unbounded ? t : unbounded;
        }
        if (key < wave_any) core.step(now, now + HALF, a.c, key + KEYS > wave_all, (int)vo_clamp64(limit - key, 0, KEYS), lane);
        unsigned char* x = now; now = next; next = x;
    }
    for (int64_t t = unbounded; t < t1; ++t) {
        vo_lds_barrier();
        fetch_k(t, now);
        vo_lds_barrier();
        const int64_t key = t * KEYS;
        if (key < wave_any) core.add_unbounded(now, vb + key * a.vs, a.vs, (int)vo_clamp64(p.Lk - key, 0, KEYS), (int)vo_clamp64(limit - key, 0, KEYS), a.c, a.D, lane);
    }
    const float l = core.across(core.l, [](float x, float y) { return x + y; });
    vo_lds_barrier();                                                // every wave is done with the key tiles
    if (a.splits > 1) {
        store_rows<float, DT>(core.o, 1.f, a.D, lds + wave * HALF, lane, [&](int r) {
            return first + r < rows ? part_row(a, split, p.q0 + token_of(first + r), head_of(first + r)) : nullptr;
        });
        if (have && lane < 32) *reinterpret_cast<float2*>(part_ml(a, split, p.q0 + token, head)) = make_float2(core.m, l);
    } else {
        store_rows<T, DT>(core.o, inverse(l), a.D, lds + wave * HALF, lane, [&](int r) {
            return first + r < rows ? out_row<T>(a, p.q0 + token_of(first + r), head_of(first + r)) : nullptr;
        });
    }
}

// ------------------------------------------------------------------------------------------------------------- rows
// A wave keeps one tile of K and one of V: the next K is requested as soon as the scores are formed, the next V after the sums, so
// one of the two is always under way.  Tiles past the end are requested too (as zeros, without any traffic): the number of
// loads under way is always the same.
template <typename T, int DT, int KEYS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attention_rows(const AttArgs a) {
    using L = Tile<T, DT>;
    constexpr int HALF = KEYS * L::ROW, MINE = 2 * HALF, PLANE = DT * 32 * 4;
    static_assert(PLANE <= MINE, "a wave's sums must fit its tiles");
    __shared__ __align__(16) unsigned char lds[WAVES * MINE];
    __shared__ float ml[WAVES][2][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned id = vo_xcd_contiguous(blockIdx.x, gridDim.x);
    const int split = id % a.splits;
    unsigned rest = id / a.splits;
    const unsigned tile = rest % a.tiles;
    const int kh = rest / a.tiles;
    const vo_place p = vo_find_tile(a.q_off, a.k_off, a.sequences, a.Tq, a.Tk, tile, a.group, 32);
    if (!p.any) return;

    const int64_t shift = p.Lk - p.Lq, rows = p.Lq * a.group;
    const int64_t last_row = p.row + 32 < rows ? p.row + 32 : rows;
    int64_t seen = a.causal ? (last_row - 1) / a.group + 1 + shift : p.Lk;
    seen = vo_clamp64(seen, 0, p.Lk);
    const int64_t key_tiles = (seen + KEYS - 1) / KEYS, per = (key_tiles + a.splits - 1) / a.splits;
    const int64_t t0 = split * per < key_tiles ? split * per : key_tiles, t1 = t0 + per < key_tiles ? t0 + per : key_tiles;

    const int64_t row = p.row + (lane & 31);
    const bool have = row < rows;
    const int64_t token = have ? row / a.group : 0;
    const int head = kh * a.group + (int)(have ? row % a.group : 0);
    Core<T, DT, KEYS> core;
    core.reset();
    core.load_q(have ? static_cast<const T*>(a.q) + (p.q0 + token) * a.qs + head * a.qh : nullptr, a.D, lane);
    const int64_t limit = a.causal ? vo_clamp64(token + shift + 1, 0, p.Lk) : p.Lk;
    int64_t all = a.causal ? vo_clamp64(p.row / a.group + shift + 1, 0, p.Lk) : p.Lk;
    if (a.vs < a.D && all == p.Lk) --all;                            // see attention_tiles

    const T* kb = static_cast<const T*>(a.k) + p.k0 * a.ks + kh * a.kh;
    const T* vb = static_cast<const T*>(a.v) + p.k0 * a.vs + kh * a.vh;
    unsigned char* mine = lds + wave * MINE;
    Loader<T, DT, KEYS, 1> lk, lv;
    lk.init(a.ks, a.D, false, 0, lane);
    lv.init(a.vs, a.D, true, 0, lane);
    unsigned char *kt = mine, *vt = mine + HALF;
    auto left = [&](int64_t t) { return t < t1 ? p.Lk - t * KEYS : 0; };
    auto fetch_k = [&](int64_t t) { lk.load(kb + t * KEYS * a.ks, a.ks, left(t), a.D, kt, 0); };
    auto fetch_v = [&](int64_t t) { lv.load(vb + t * KEYS * a.vs, a.vs, left(t), a.D, vt, 0); };
    constexpr int N = Loader<T, DT, KEYS, 1>::N;
    static_assert(N < 64, "the counter has six bits");
    auto arrived = [] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); };          // all but the N youngest loads
    auto consumed = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };                // a tile's reads, before it is loaded over
    if (t0 + wave < t1) {
        fetch_k(t0 + wave);
        fetch_v(t0 + wave);
    }
    int64_t unbounded = t1;                                          // the wave's first tile that was bounded
    for (int64_t t = t0 + wave; t < t1; t += WAVES) {
        const int64_t key = t * KEYS;
        vo_f32x16 s[core.KB];
        unsigned w[core.KB][core.PW];
        arrived();
        core.scores(kt, s, lane);
        consumed();
        fetch_k(t + WAVES);
        if (key + KEYS > all) core.mask(s, (int)vo_clamp64(limit - key, 0, KEYS), lane);
        core.follow(core.largest(s), a.c);
        core.weights(s, w, a.c);
        arrived();
        if (key + KEYS > all && all < p.Lk && core.any_unbounded(vt, lane)) {
            core.bound(vt, 0, 1, lane);
            vo_wave_lds_fence();
            unbounded = t < unbounded ? t : unbounded;
        }
        core.accumulate(vt, w, lane);
        consumed();
        fetch_v(t + WAVES);
    }
    for (int64_t t = unbounded; t < t1; t += WAVES) {
        const int64_t key = t * KEYS;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // nothing is under way into the tile or read from it
        fetch_k(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        core.add_unbounded(kt, vb + key * a.vs, a.vs, (int)vo_clamp64(p.Lk - key, 0, KEYS), (int)vo_clamp64(limit - key, 0, KEYS), a.c, a.D, lane);
    }
    core.l = core.across(core.l, [](float x, float y) { return x + y; });

    // Join the waves in order: sums as (feature, row) planes over the wave's own tiles, where nothing is under way any more.  Features
    // four apart (the two halves of a wave) change places with a neighbour so that they meet other banks.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    auto at = [&](int f) { return (f ^ (f >> 2 & 1)) * 32 + (lane & 31); };
    float* sums = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[at(d * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3))] = core.o[d][i];
    if (lane < 32) {
        ml[wave][0][lane] = core.m;
        ml[wave][1][lane] = core.l;
    }
    __syncthreads();
    float w[WAVES], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, ml[i][0][lane & 31]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        w[i] = m == -INFINITY ? 0.f : exp2f((ml[i][0][lane & 31] - m) * a.c);
        l += w[i] * ml[i][1][lane & 31];
    }
    // eight features, four to each half of the wave, at a time: wave w takes the pieces w, w + WAVES, ..
    const float inv = inverse(l);
    for (int piece = wave; piece < DT / 8; piece += WAVES) {
        const int f = piece * 8 + 4 * (lane >> 5);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) v[j] += w[i] * reinterpret_cast<const float*>(lds + i * MINE)[at(f + j)];
        }
        if (!have || f >= a.D) continue;
        if (a.splits > 1) {
            *reinterpret_cast<vo_f32x4*>(part_row(a, split, p.q0 + token, head) + f) = vo_f32x4{v[0], v[1], v[2], v[3]};
        } else if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<vo_u32x2*>(out_row<T>(a, p.q0 + token, head) + f) =
                vo_u32x2{vo_elem<T>::pack2(in_range<T>(v[0] * inv), in_range<T>(v[1] * inv)), vo_elem<T>::pack2(in_range<T>(v[2] * inv), in_range<T>(v[3] * inv))};
        } else {
            *reinterpret_cast<vo_f32x4*>(out_row<T>(a, p.q0 + token, head) + f) = vo_f32x4{v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        }
    }
    if (a.splits > 1 && wave == 0 && lane < 32 && have)
        *reinterpret_cast<float2*>(part_ml(a, split, p.q0 + token, head)) = make_float2(m, l);
}

// ------------------------------------------------------------------------------------------------------------- join
// One wave per (token, head): lane s takes the weight of part s; then groups of WIDTH lanes, four features a lane, each add every
// (64 / WIDTH)-th part, and the groups' sums are added crosswise: a fixed order.  Rows outside every sequence stay as they are.
template <typename T, int WIDTH> __global__ __launch_bounds__(256) void attention_join(const AttArgs a) {
    constexpr int GROUPS = 64 / WIDTH;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t token = row / a.Hq;
    if (token >= a.Tq) return;
    if (a.q_off && (token < a.q_off[0] || token >= a.q_off[a.sequences])) return;
    const int head = (int)(row % a.Hq), f = lane % WIDTH * 4;
    // a round's sums are requested before the weights are known: a part is written for every row of a sequence
    vo_f32x4 x[4];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * GROUPS + lane / WIDTH;
            x[i] = vo_f32x4{0.f, 0.f, 0.f, 0.f};
            if (s < a.splits && f < a.D) x[i] = *reinterpret_cast<const vo_f32x4*>(part_row(a, s, token, head) + f);
        }
    };
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < a.splits) ml = *reinterpret_cast<const float2*>(part_ml(a, lane, token, head));
    fetch(0);
    float m = ml.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float w = ml.x == -INFINITY ? 0.f : exp2f((ml.x - m) * a.c);
    float l = w * ml.y;                                              // a part that saw no key of this row has neither weight nor sums
#pragma unroll
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += 4 * GROUPS) {
        if (s0) fetch(s0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float ws = __shfl(w, s0 + i * GROUPS + lane / WIDTH & 63);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += ws * x[i][j];
        }
    }
#pragma unroll
    for (int d = 32; d >= WIDTH; d >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], d);
    if (lane >= WIDTH || f >= a.D) return;
    const float inv = inverse(l);
    T* p = out_row<T>(a, token, head) + f;
#pragma unroll
    for (int j = 0; j < 4; ++j) vo_elem<T>::put(p + j, in_range<T>(o[j] * inv));
}

// ------------------------------------------------------------------------------------------------------------- host

struct Plan {
    bool rows;
    int splits;
    int64_t tiles, blocks;
};

// The features that a head is padded to, keys in a tile and workgroups a CU holds (LDS and registers) in the form by tiles.
// 96 features: 16 heads of 72 or 96 over 4, 4 sequences of 3000, take 144 and 148 us, padded to 128 186 and 192.  32 keys in
// float32, whose values take twice the registers, for more workgroups: 4800 rows, 4 heads of 64: 204 us, with 64 keys 226; 3000 rows,
// 8 heads of 128 over 2, causal: 196, with 64 keys and one workgroup a CU 424.
constexpr int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256; }
constexpr int tile_keys(int DT, int es) { return DT * es > 512 || (es == 4 && DT >= 64) ? 32 : 64; }
constexpr int rows_waves(int DT, int es) { return DT * es <= 256 ? 8 : DT * es <= 512 ? 4 : 2; }
constexpr int tile_blocks(int DT) { return DT <= 64 ? 4 : DT == 96 ? 3 : DT == 128 ? 2 : 1; }

// The lengths are on the device, so the averages decide.  What that costs where they differ much (bfloat16, 32 heads over 8 of 128, causal):
// single rows, a history of 32768 keys among 63 of 100: 186 us, in two calls 47; a prompt of 4096 among 600 tokens before 100 keys: 408
// and 296; among 20 tokens before 2000 keys: 158 and 182.
Plan plan(int64_t Tq, int64_t Tk, int sequences, int Hq, int Hk, int D, int dtype) {
    const int group = Hq / Hk;
    Plan p{};
    const int64_t rows = vo_ceil_div(Tq * group, sequences);         // a sequence's rows per key head, on average
    const int64_t keys = vo_ceil_div(Tk, sequences);
    p.rows = rows <= 32;
    p.tiles = vo_tiles_bound(Tq, sequences, group, p.rows ? 32 : 128);
    const int64_t base = p.tiles * Hk;
    int64_t splits = 1;
    if (p.rows) {
        // Few workgroups: parts until every CU has one (and none two: that round would be as long again), of at least 256 keys, where
        // the join's launch is worth it (one row before 777 keys, 8 key heads: 12.2 us unsplit, 12.0 in 4 parts; 1500 keys: 16.1 /
        // 12.7; 4096: 33.0 / 18.0, 14.3 in 16).
        if (keys >= 1024) {
            splits = 256 / base;
            if (splits > keys / 256) splits = keys / 256;
        }
        // Many: about eight rounds over the CUs even out sequences of different lengths, but parts under 2048 keys cost more than that
        // gains (32 sequences of up to 32768 keys: 501 us unsplit, 400 in 4 parts, 383 in 8, 409 in 16; 64 of 2000: 111, 135 in 4).
        const int64_t even = vo_ceil_div(2048, base) < keys / 2048 ? vo_ceil_div(2048, base) : keys / 2048;
        if (splits < even) splits = even;
    } else {
        // Rounds over the resident workgroups times a part's key tiles and its start, plus the join's traffic.  (One sequence of
        // 4800 float32 rows, 4 heads of 64: 357 us unsplit, 224 in 3 parts, 249 in 4, 213 in 5, 222 in 8; 96 rows before 30001 keys, 32
        // heads over 4: 518 unsplit, 100 in 10, 78 in 18, 85 in 32.)
        const int es = dtype == VO_F32 ? 4 : 2, tile = tile_keys(padded(D), es);
        const int64_t resident = 256 * tile_blocks(padded(D));
        // In float32 the products alone take the time, whichever workgroup of a CU they belong to: 2 x keys x features cycles a tile.
        // The lengths are on the device: where all workgroups run at once, the longest sequence, taken to be half as long again as the
        // average, is what they wait for (8 sequences of 71 to 1500 keys: 26 us unsplit, 16 in 4 parts; 2 equal ones of 20000 keys
        // lose 5 %).
        const int64_t longest = keys + keys / 2 < Tk ? keys + keys / 2 : Tk;
        const double tiles = (double)vo_ceil_div(keys, tile), most = (double)vo_ceil_div(longest, tile), tile_us = D / 128.0 * 2.1;
        const double join_us = (double)Tq * Hq * D * 8 / 4e6;        // per part: written and read once
        double best = 0.;
        for (int s = 1; s <= 64 && s <= (longest + 255) / 256; ++s) {
            const double blocks = (double)base * s, rounds = blocks <= resident ? 0.6 + 0.4 * blocks / resident : (double)((int64_t)((blocks + resident - 1) / resident));
            double us = rounds * ((blocks <= resident ? most : tiles) / s + 2.) * tile_us;
            if (dtype == VO_F32) us = (double)vo_ceil_div(base * s, 256) * (most / s + 2.) * tile * padded(D) / 980.;
            if (s > 1) us += 4. + s * join_us;
            if (s == 1 || us < best) {
                best = us;
                splits = s;
            }
        }
    }
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
    p.splits = (int)splits;
    p.blocks = base * splits;
    return p;
}

// A launch has fewer than 2^32 threads.  Sizes that pass this by far (2^25 workgroups of the fewest threads, by a bound from below) are
// told first: the products in plan() could pass 64 bits.
bool too_many(int64_t Tq, int sequences, int Hq, int Hk) { return (double)Tq * Hq / 128 + (sequences - 1.) * Hk >= (double)(1 << 25); }
bool too_many(const Plan& p, int64_t Tq, int Hq, int D, int dtype) {
    const int threads = p.rows ? 64 * rows_waves(padded(D), dtype == VO_F32 ? 4 : 2) : 256;
    return p.blocks * threads >= (1ll << 32) || (p.splits > 1 && Tq * Hq * 64 >= (1ll << 32));
}

int64_t workspace(const Plan& p, int64_t Tq, int Hq, int D) { return p.splits > 1 ? (int64_t)p.splits * Tq * Hq * (D + 2) * 4 : 0; }

template <typename T, int DT> int launch(const AttArgs& a, const Plan& p, hipStream_t st) {
    constexpr int BYTES = DT * (int)sizeof(T);                       // of a row
    const dim3 grid((unsigned)p.blocks);
    if (p.rows) {
        constexpr int KEYS = BYTES <= 128 ? 64 : 32, WAVES = rows_waves(DT, sizeof(T));
        attention_rows<T, DT, KEYS, WAVES><<<grid, 64 * WAVES, 0, st>>>(a);
    } else {
        attention_tiles<T, DT, tile_keys(DT, sizeof(T)), tile_blocks(DT)><<<grid, 256, 0, st>>>(a);
    }
    VO_CHECK_LAUNCH("vo_attention");
    if (p.splits > 1) {
        attention_join<T, DT == 96 ? 32 : DT / 4><<<dim3((unsigned)vo_ceil_div(a.Tq * a.Hq, 4)), 256, 0, st>>>(a);
        VO_CHECK_LAUNCH("vo_attention (join)");
    }
    return VO_OK;
}

template <typename T> int dispatch(const AttArgs& a, const Plan& p, hipStream_t st) {
    if (a.D <= 32) return launch<T, 32>(a, p, st);
    if (a.D <= 64) return launch<T, 64>(a, p, st);
    if (a.D <= 96) return launch<T, 96>(a, p, st);
    if (a.D <= 128) return launch<T, 128>(a, p, st);
    return launch<T, 256>(a, p, st);
}

}  // namespace

extern "C" int64_t vo_attention_workspace_bytes(int64_t q_tokens, int64_t k_tokens, int sequences, int q_heads, int k_heads, int D, int dtype) {
    if (q_tokens <= 0 || k_tokens < 0 || sequences <= 0 || q_heads <= 0 || k_heads <= 0 || q_heads % k_heads || D <= 0) return 0;
    if (too_many(q_tokens, sequences, q_heads, k_heads)) return 0;
    return workspace(plan(q_tokens, k_tokens, sequences, q_heads, k_heads, D, dtype), q_tokens, q_heads, D);
}

extern "C" int vo_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                            int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, void* out,
                            int64_t out_token_stride, int64_t out_head_stride, const int32_t* q_offsets, const int32_t* k_offsets,
                            int sequences, int64_t q_tokens, int64_t k_tokens, int q_heads, int k_heads, int D, float scale, int causal,
                            int dtype, void* workspace_ptr, int64_t workspace_bytes, void* stream) {
    VO_REQUIRE(dtype == VO_F32 || dtype == VO_F16 || dtype == VO_BF16, "vo_attention: dtype=%d is none of VO_F32, VO_F16, VO_BF16", dtype);
    VO_REQUIRE(sequences >= 1 && q_tokens >= 0 && k_tokens >= 0 && q_heads >= 1 && k_heads >= 1 && q_heads % k_heads == 0,
               "vo_attention: sequences=%d q_tokens=%lld k_tokens=%lld heads %d / %d (heads a multiple of the key heads)", sequences,
               (long long)q_tokens, (long long)k_tokens, q_heads, k_heads);
    VO_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "vo_attention: scale must be positive (1e-30 to 1e30)");
    VO_REQUIRE((q_offsets && k_offsets) || (!q_offsets && !k_offsets && sequences == 1),
               "vo_attention: both offset arrays, or none and one sequence");
    const int64_t es = dtype == VO_F32 ? 4 : 2;
    if (D < 1 || D > 256 || D * es % 16) return vo_fail(VO_ERR_UNSUPPORTED, "vo_attention: D=%d must be at most 256 and whole 16-byte pieces", D);
    if (q_tokens == 0) return VO_OK;
    VO_REQUIRE(q && out && (k_tokens == 0 || (k && v)), "vo_attention: null pointer");
    // a key tile is addressed with 32-bit offsets from its first token; heads are 64-bit products
    const int64_t strides[] = {q_token_stride, k_token_stride, v_token_stride, out_token_stride, q_head_stride, k_head_stride, v_head_stride, out_head_stride};
    for (int i = 0; i < 8; ++i) {
        const int64_t s = strides[i];
        if (s < 0 || s % (16 / es) || (i < 4 && s >= (1ll << 24) / es))
            return vo_fail(VO_ERR_UNSUPPORTED, "vo_attention: strides must be whole 16-byte pieces, tokens' under 16 MiB (got %lld elements between %s)",
                           (long long)s, i < 4 ? "tokens" : "heads");
    }
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) % 16)
        return vo_fail(VO_ERR_UNSUPPORTED, "vo_attention: tensors must be 16-byte aligned");
    if (q_tokens >= (1ll << 31) || k_tokens >= (1ll << 31))
        return vo_fail(VO_ERR_UNSUPPORTED, "vo_attention: offsets are 32-bit: fewer than 2^31 tokens");
    const bool many = too_many(q_tokens, sequences, q_heads, k_heads);
    const Plan p = many ? Plan{} : plan(q_tokens, k_tokens, sequences, q_heads, k_heads, D, dtype);
    if (many || too_many(p, q_tokens, q_heads, D, dtype))
        return vo_fail(VO_ERR_UNSUPPORTED, "vo_attention: %lld tokens of %d heads are too many for one launch", (long long)q_tokens, q_heads);
    const int64_t need = workspace(p, q_tokens, q_heads, D);
    VO_REQUIRE(need == 0 || (workspace_ptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace_ptr) % 16 == 0),
               "vo_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    AttArgs a{};
    a.q = q; a.k = k; a.v = v; a.out = out; a.part = static_cast<float*>(workspace_ptr);
    a.q_off = q_offsets; a.k_off = k_offsets;
    a.qs = q_token_stride; a.qh = q_head_stride; a.ks = k_token_stride; a.kh = k_head_stride;
    a.vs = v_token_stride; a.vh = v_head_stride; a.os = out_token_stride; a.oh = out_head_stride;
    a.Tq = q_tokens; a.Tk = k_tokens;
    a.sequences = sequences; a.Hq = q_heads; a.Hk = k_heads; a.group = q_heads / k_heads;
    a.D = D; a.causal = causal != 0; a.splits = p.splits;
    a.tiles = (unsigned)p.tiles;
    a.reciprocal = a.group <= 128 ? (65535u + a.group) / a.group : 0;
    a.c = scale * LOG2E;
    hipStream_t st = vo_stream(stream);
    if (dtype == VO_F32) return dispatch<float>(a, p, st);
    if (dtype == VO_F16) return dispatch<_Float16>(a, p, st);
    return dispatch<__bf16>(a, p, st);
}
