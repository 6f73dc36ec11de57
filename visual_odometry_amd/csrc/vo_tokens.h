// Shared pieces of the token-major operators (vo_linear.hip, vo_attention.hip): element types, 16-byte chunks of a row
// and the matrix instruction on them.  gfx950 only.
#pragma once

#include "vo_common.h"

typedef unsigned vo_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned vo_u32x2 __attribute__((ext_vector_type(2)));
typedef float vo_f32x4 __attribute__((ext_vector_type(4)));
typedef float vo_f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 vo_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 vo_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 vo_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 vo_bf16x2 __attribute__((ext_vector_type(2)));

// One row's 16 bytes (`PER` elements) as a matrix operand.  In every 16x16 product below lane l brings row l % 16 of each
// operand and the chunk number l / 16 of it, so the four lane groups cover 4 * PER consecutive elements of the summed axis;
// in a 32x32 product row l % 32 and chunk l / 32.  Which element of the sum meets which lane does not matter as long as
// both operands agree, which is what makes the float32 form (one element per lane and instruction) read the same chunks.
// Result: column (second operand's row) l % 16, rows (first operand's) 4 * (l / 16) + i; of the 32x32 form column l % 32,
// rows 8 * (i / 4) + 4 * (l / 32) + i % 4.
template <typename T> struct vo_elem;

template <> struct vo_elem<float> {
    static constexpr int PER = 4;
    static constexpr int PARTS = 4;                                  // instructions per chunk: callers put other sums between them
    static __device__ __forceinline__ vo_f32x4 mma16(vo_u32x4 a, vo_u32x4 b, vo_f32x4 c, int part) {
        const vo_f32x4 x = __builtin_bit_cast(vo_f32x4, a), y = __builtin_bit_cast(vo_f32x4, b);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(x[part], y[part], c, 0, 0, 0);
    }
    static __device__ __forceinline__ vo_f32x16 mma32(vo_u32x4 a, vo_u32x4 b, vo_f32x16 c, int part) {
        const vo_f32x4 x = __builtin_bit_cast(vo_f32x4, a), y = __builtin_bit_cast(vo_f32x4, b);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(x[part], y[part], c, 0, 0, 0);
    }
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(vo_u32x4 r, float* v) {
        const vo_f32x4 t = __builtin_bit_cast(vo_f32x4, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = t[j];
    }
    static __device__ __forceinline__ vo_u32x4 pack(const float* v) {
        return __builtin_bit_cast(vo_u32x4, vo_f32x4{v[0], v[1], v[2], v[3]});
    }
};

// The 16-bit types: products are exact in the accumulator's float32, a value is rounded (to nearest even) only where a
// result leaves in the tensor's type.
template <> struct vo_elem<_Float16> {
    static constexpr int PER = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ vo_f32x4 mma16(vo_u32x4 a, vo_u32x4 b, vo_f32x4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vo_f16x8, a), __builtin_bit_cast(vo_f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ vo_f32x16 mma32(vo_u32x4 a, vo_u32x4 b, vo_f32x16 c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vo_f16x8, a), __builtin_bit_cast(vo_f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float get(const _Float16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }
    static __device__ __forceinline__ unsigned pack2(float a, float b) {
        vo_f16x2 t; t[0] = (_Float16)a; t[1] = (_Float16)b;
        return __builtin_bit_cast(unsigned, t);
    }
    static __device__ __forceinline__ void unpack(vo_u32x4 r, float* v) {
        const vo_f16x8 t = __builtin_bit_cast(vo_f16x8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
    }
    static __device__ __forceinline__ vo_u32x4 pack(const float* v) {
        return vo_u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
    }
};

template <> struct vo_elem<__bf16> {
    static constexpr int PER = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ vo_f32x4 mma16(vo_u32x4 a, vo_u32x4 b, vo_f32x4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vo_bf16x8, a), __builtin_bit_cast(vo_bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ vo_f32x16 mma32(vo_u32x4 a, vo_u32x4 b, vo_f32x16 c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vo_bf16x8, a), __builtin_bit_cast(vo_bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float get(const __bf16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(__bf16* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ unsigned pack2(float a, float b) {
        vo_bf16x2 t; t[0] = (__bf16)a; t[1] = (__bf16)b;
        return __builtin_bit_cast(unsigned, t);
    }
    static __device__ __forceinline__ void unpack(vo_u32x4 r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __builtin_bit_cast(float, r[j] << 16);
            v[2 * j + 1] = __builtin_bit_cast(float, r[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ vo_u32x4 pack(const float* v) {
        return vo_u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
    }
};

// Buffer descriptor over `bytes` from p: loads behind it return 0 and stores behind it are dropped, so tile edges need no
// branches.  An offset of VO_OUTSIDE is behind every descriptor (they span less than 2 GiB), also with some MiB added to it.
// The whole offset goes into the lane's own operand: the range check subtracts the scalar operand from the size and would
// wrap around where that operand is the larger.
constexpr unsigned VO_OUTSIDE = 0x80000000u;
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t vo_buffer(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// 16 bytes per lane from a buffer straight into LDS: lane l's bytes land at lds + 16 * l (lds is wave-uniform).
static __device__ __forceinline__ void vo_load_to_lds(__amdgpu_buffer_rsrc_t rs, void* lds, unsigned offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
}

// Waits for this wave's loads into LDS and its LDS reads, then for the workgroup.  Spelled out because the compiler's own
// barrier does not count loads into LDS in every loop (another wave's load was read too early without it), and would not
// leave any pending.
// PENDING: how many of this wave's youngest loads may still be under way.
template <int PENDING = 0> static __device__ __forceinline__ void vo_lds_barrier() {
    static_assert(PENDING >= 0 && PENDING < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");
}

// 16 bytes at any address: the memory pipes take unaligned accesses, the compiler just has to be told.
static __device__ __forceinline__ vo_u32x4 vo_load16(const void* p) {
    vo_u32x4 r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
static __device__ __forceinline__ void vo_store16(void* p, vo_u32x4 v) { __builtin_memcpy(p, &v, 16); }

// 16 bytes moved down by 0 to 15 bytes, zeros behind.
static __device__ __forceinline__ vo_u32x4 vo_move_down(vo_u32x4 r, int bytes) {
    const int bits = bytes * 8;
    uint64_t lo = (uint64_t)r[1] << 32 | r[0], hi = (uint64_t)r[3] << 32 | r[2];
    if (bits >= 64) {
        lo = hi >> (bits - 64);
        hi = 0;
    } else if (bits > 0) {
        lo = lo >> bits | hi << (64 - bits);
        hi >>= bits;
    }
    return vo_u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}

// PER elements of a row from p on, which may have any address; `n` of them exist (the others become zero) and `before` elements of
// the row lie ahead of p.  A row's last, shorter piece is the row's last 16 bytes moved down.
template <typename T> static __device__ __forceinline__ vo_u32x4 vo_load_unaligned(const T* p, int64_t n, int64_t before) {
    constexpr int PER = vo_elem<T>::PER;
    vo_u32x4 r = {0, 0, 0, 0};
    if (n >= PER) {
        r = vo_load16(p);
    } else if (n > 0 && n + before >= PER) {
        r = vo_move_down(vo_load16(p - (PER - n)), (PER - (int)n) * (int)sizeof(T));
    } else if (n > 0) {
        float v[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = j < n ? vo_elem<T>::get(p + j) : 0.f;
        r = vo_elem<T>::pack(v);                                      // exact: the values come from the type itself
    }
    return r;
}

// A workgroup's number among `total` renumbered so that the workgroups of one XCD (they are dealt out round robin over the
// eight) get consecutive numbers: neighbours share operands in that XCD's L2.
static __device__ __forceinline__ unsigned vo_xcd_contiguous(unsigned id, unsigned total) {
    const unsigned per = total / 8, rest = total % 8, xcd = id % 8, i = id / 8;
    return xcd * per + (xcd < rest ? xcd : rest) + i;
}

// Orders this wave's LDS writes before its later LDS reads of other lanes' values (no other wave involved).
static __device__ __forceinline__ void vo_wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
