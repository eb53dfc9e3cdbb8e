// What the language-model operators share: 16-bit types and their matrix products, loads from memory straight into LDS, transposed
// LDS reads, exchanges between the halves of a wave. gfx950 only.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace lm {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Operands travel as eight 16-bit patterns (s16x8), whatever they stand for; Type says how they are multiplied and rounded.
struct Bf16 {
    typedef bf16_t value;
    static constexpr bool wide_range = true; // exponents of 32 bits: gradients need no scale
    static constexpr short EXPONENT = 0x7f80;
    static __device__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c)
    {
        typedef bf16_t v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};
struct F16 {
    typedef f16_t value;
    static constexpr bool wide_range = false;
    static constexpr short EXPONENT = 0x7c00;
    static __device__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c)
    {
        typedef f16_t v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};

template <class Type>
__device__ inline short to16(float x)
{
    return __builtin_bit_cast(short, static_cast<typename Type::value>(x));
}
template <class Type>
__device__ inline float to32(short x)
{
    return static_cast<float>(__builtin_bit_cast(typename Type::value, x));
}

typedef __attribute__((address_space(3))) void lds_void;
typedef __amdgpu_buffer_rsrc_t buffer_t;

// A window of memory whose reads past `bytes` give zeros and touch nothing.
__device__ inline buffer_t window(const void* base, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00020000);
}
constexpr uint32_t OUTSIDE = 0x80000000u; // an offset that no window reaches: windows hold less than 2^31 bytes

// 16 bytes a lane from the window to LDS, lane l's at dst + 16 l; arrives before the wave's next wait for its loads.
__device__ inline void load_to_lds(buffer_t w, void* dst, uint32_t offset)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (lds_void*)dst, 16, static_cast<int>(offset), 0, 0, 0);
}

__device__ inline s16x8 read16(const short* p) { return *reinterpret_cast<const s16x8*>(p); }

// A 4 x 16 block per 16 lanes, turned: lane j of a group names the j-th run of four of the block's sixteen (row j / 4, columns
// 4 (j % 4) ...) and gets column j, rows 0 to 3.
__device__ inline s16x4 read_turned(const short* p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
__device__ inline s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// What lane l ^ 32 holds.
__device__ inline float other_half(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, threadIdx.x & 32 ? r[0] : r[1]);
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;


__device__ inline void wait_for_all() { __builtin_amdgcn_s_waitcnt(0x0070); } // loads and LDS accesses: vmcnt(0), lgkmcnt(0)
__device__ inline void wait_for_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); } // LDS accesses alone: lgkmcnt(0)
// All waves of the workgroup, without a wait for loads in flight; the compiler moves no memory access across it.
__device__ inline void meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

} // namespace lm
