// Packed sequences cut into row tiles, without any length known to the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// Where a row tile lies.  Sequence s owns the tiles from first_tile(s) = rows before it / tile size + s on: that leaves every
// sequence at least the tiles it needs (floor(b/T) - floor(a/T) + 1 >= ceil((b - a)/T)), so a tile finds its sequence by a
// search: a wave tests 64 candidates at once (bisection's ten dependent loads for a thousand sequences were a good part of a
// short sequence's time).
struct vo_place {
    int64_t q0, k0;                               // the sequence's first row (token) and key
    int64_t Lq, Lk;
    int64_t row;                                  // first row of the tile within the sequence (rows_per_token rows a token)
    bool any;                                     // the tile holds a row
};

__host__ __device__ inline int64_t vo_clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// Tiles of all sequences together: an upper bound.
__host__ __device__ inline int64_t vo_tiles_bound(int64_t tokens, int sequences, int rows_per_token, int rows_per_tile) {
    return tokens * rows_per_token / rows_per_tile + sequences;
}

// Offsets are clamped to the tensors, so wrong ones cannot lead outside them.  No offsets: one sequence of everything.
__host__ __device__ inline vo_place vo_find_tile(const int* q_off, const int* k_off, int sequences, int64_t q_tokens, int64_t k_tokens,
                                                 unsigned tile, int rows_per_token, int rows_per_tile) {
    vo_place p;
    int s = 0;
    p.q0 = 0;
    p.Lq = q_tokens;
    p.k0 = 0;
    p.Lk = k_tokens;
    if (q_off) {
        int hi = sequences;                       // first_tile(s) <= tile < first_tile(hi), but for s = 0 and hi = sequences
        while (hi - s > 1) {
            const int step = (hi - s + 63) / 64;  // candidates s + step, s + 2 step, ..: how many of them start at or before the tile?
            auto before = [&](int i) {
                const int64_t c = s + (int64_t)(i + 1) * step;
                return c < hi && vo_clamp64(q_off[c], 0, q_tokens) * rows_per_token / rows_per_tile + c <= tile;
            };
            int n = 0;
#ifdef __HIP_DEVICE_COMPILE__
            n = __builtin_popcountll(__ballot(before(threadIdx.x & 63)));
#else
            for (int i = 0; i < 64; ++i) n += before(i);
#endif
            s += n * step;
            if (s > hi - 1) s = hi - 1;           // only offsets that do not ascend lead there
            if (hi > s + step) hi = s + step;
        }
        p.q0 = vo_clamp64(q_off[s], 0, q_tokens);
        p.Lq = vo_clamp64(q_off[s + 1], p.q0, q_tokens) - p.q0;
        p.k0 = vo_clamp64(k_off[s], 0, k_tokens);
        p.Lk = vo_clamp64(k_off[s + 1], p.k0, k_tokens) - p.k0;
    }
    p.row = ((int64_t)tile - (p.q0 * rows_per_token / rows_per_tile + s)) * rows_per_tile;
    p.any = p.row >= 0 && p.row < p.Lq * rows_per_token;
    return p;
}
