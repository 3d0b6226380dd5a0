// The 8-bit block format shared by the fp8 kernels.
//
// A row of C elements is cut into blocks of 128 (the last one may be shorter).  A block is stored as one byte per
// element (OCP e4m3 or e5m2) and one scale byte s = e + 127 standing for 2^e, where e is the smallest integer >= -126
// with amax <= MAX * 2^e and amax is the largest FINITE magnitude of the block (a block without one has e = 0).
// An element is round_to_nearest_even(x * 2^-e): the product is exact up to underflow far below the smallest 8-bit
// step, so x is rounded once.  NaN stays NaN; an infinity becomes NaN in e4m3, which has none, and stays one in e5m2.
// The scale is a power of two because the matrix instruction applies such scales itself (E8M0 operands of
// v_mfma_scale_f32_16x16x128_f8f6f4, whose reduction length is exactly one block): no multiplication is left for the
// vector unit, and bf16 holds every restored value exactly (4 significant bits at most; of blocks with scales under 2^-124, e5m2
// 2^-117, the smallest elements are rounded to its smallest step, 2^-133).
// Rows of bytes are padded with zeros to whole 16-byte pieces, rows of scales with 127 to whole groups of four.
#pragma once
#include "mma.h"

namespace mad {

constexpr int F8_BLOCK = 128;
constexpr int F8_E4M3 = 0, F8_E5M2 = 1;      // also the matrix instruction's operand type codes

__host__ __device__ __forceinline__ int f8_pitch(int C) { return (C + 15) & ~15; }
__host__ __device__ __forceinline__ int f8_blocks(int C) { return (C + F8_BLOCK - 1) / F8_BLOCK; }
__host__ __device__ __forceinline__ int f8_scale_pitch(int C) { return (f8_blocks(C) + 3) & ~3; }

// packed parts lie where their wide accesses need them
inline bool f8_aligned(const void* q, const void* scale) { return !((uintptr_t)q & 15) && !((uintptr_t)scale & 3); }

// bits of |x|, 0 for a value that is not finite: their unsigned maximum is the block's amax
__device__ __forceinline__ unsigned f8_mag(float x) {
    const unsigned u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// scale byte of a block from the bits of its amax: MAX = 1.75 * 2^8 (e4m3), 1.75 * 2^15 (e5m2)
template <int FMT> __device__ __forceinline__ unsigned f8_scale_byte(unsigned amax) {
    int s = (int)(amax >> 23) - (FMT == F8_E4M3 ? 8 : 15) + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    s = s < 1 ? 1 : s;
    return amax ? (unsigned)s : 127u;
}
__device__ __forceinline__ float f8_scale(unsigned byte) { return __uint_as_float(byte << 23); }            // 2^e
__device__ __forceinline__ float f8_inv_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }  // 2^-e

template <int FMT> __device__ __forceinline__ unsigned f8_cvt4(float a, float b, float c, float d) {
    int r;
    if (FMT == F8_E4M3) {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    } else {
        r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
        r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
    }
    return (unsigned)r;
}

// Four bf16 (two dwords) times 2^-e as four bytes, one instruction per pair.  The conversion divides by its scale operand, whose
// exponent alone counts: scale is 2^e.
template <int FMT> __device__ __forceinline__ unsigned f8_cvt4_bf16(unsigned lo, unsigned hi, float scale) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 r = {0, 0};
    if (FMT == F8_E4M3) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, lo), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, hi), scale, true);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(r, __builtin_bit_cast(bf16x2, lo), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(r, __builtin_bit_cast(bf16x2, hi), scale, true);
    }
    return __builtin_bit_cast(unsigned, r);
}

// the four values of one dword, times 2^e
template <int FMT> __device__ __forceinline__ void f8_values4(unsigned q, float scale, float* f) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    f32x2 lo, hi;
    if (FMT == F8_E4M3) {
        lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false);
        hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    } else {
        lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)q, false);
        hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)q, true);
    }
    f[0] = lo[0] * scale; f[1] = lo[1] * scale; f[2] = hi[0] * scale; f[3] = hi[1] * scale;
}

// eight bytes times a power of two as bf16: exact (4 significant bits) down to bf16's smallest step
template <int FMT> __device__ __forceinline__ bf16x8 f8_bf16x8(unsigned lo, unsigned hi, float scale = 1.0f) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 a, b, c, d;
    if (FMT == F8_E4M3) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false); b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false); d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, false); b = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, false); d = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, true);
    }
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// unsigned maximum over the 16 lanes of a row of lanes (every lane receives it)
__device__ __forceinline__ unsigned row16_umax(unsigned v) {
    auto step = [](unsigned a, unsigned b) { return a > b ? a : b; };
    v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));     // lane ^ 1
    v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));     // lane ^ 2
    v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));    // mirror of 8
    v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));    // mirror of 16
    return v;
}

// Eight consecutive elements at any element-aligned address (rows of odd length start anywhere).
template <typename T> __device__ __forceinline__ void load8(const T* p, float* f);
template <> __device__ __forceinline__ void load8<bf16_t>(const bf16_t* p, float* f) {
    typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    const u32x4u v = *reinterpret_cast<const u32x4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(v[i] << 16); f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float* f) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const f32x4u a = reinterpret_cast<const f32x4u*>(p)[0], b = reinterpret_cast<const f32x4u*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f);
template <> __device__ __forceinline__ void store8<bf16_t>(bf16_t* p, const float* f) {
    typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    u32x4u v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (unsigned)f32_to_bf16(f[2 * i]) | ((unsigned)f32_to_bf16(f[2 * i + 1]) << 16);
    *reinterpret_cast<u32x4u*>(p) = v;
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float* f) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    reinterpret_cast<f32x4u*>(p)[0] = f32x4u{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4u*>(p)[1] = f32x4u{f[4], f[5], f[6], f[7]};
}
// eight elements as they were loaded (their conversion waits until they are added)
template <typename T> struct Piece8;
template <> struct Piece8<bf16_t> {
    typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    u32x4u v;
    __device__ __forceinline__ void load(const bf16_t* p) { v = *reinterpret_cast<const u32x4u*>(p); }
    __device__ __forceinline__ void add(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] += __uint_as_float(v[i] << 16); f[2 * i + 1] += __uint_as_float(v[i] & 0xffff0000u); }
    }
};
template <> struct Piece8<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) { load8<float>(p, v); }
    __device__ __forceinline__ void add(float* f) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += v[i];
    }
};
// the same for a piece that may reach past column C (columns behind it read as zero, are not written)
template <typename T> __device__ __forceinline__ void load8_tail(const T* p, int c, int C, float* f) {
    if (c + 8 <= C) { load8<T>(p, f); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < C ? Elem<T>::load(p[i]) : 0.0f;
}
template <typename T> __device__ __forceinline__ void store8_tail(T* p, int c, int C, const float* f) {
    if (c + 8 <= C) { store8<T>(p, f); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) if (c + i < C) p[i] = Elem<T>::store(f[i]);
}

// four consecutive elements, likewise
template <typename T> __device__ __forceinline__ void store4_tail(T* p, int c, int C, const f32x4& f) {
    if (c + 4 <= C) {
        if constexpr (sizeof(T) == 2) {
            typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
            *reinterpret_cast<u32x2u*>(p) = u32x2u{(unsigned)f32_to_bf16(f[0]) | ((unsigned)f32_to_bf16(f[1]) << 16),
                                                   (unsigned)f32_to_bf16(f[2]) | ((unsigned)f32_to_bf16(f[3]) << 16)};
        } else {
            typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<f32x4u*>(p) = f;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (c + i < C) p[i] = Elem<T>::store(f[i]);
}
template <typename T> __device__ __forceinline__ f32x4 load4_tail(const T* p, int c, int C) {
    f32x4 f = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c + 4 <= C) {
        if constexpr (sizeof(T) == 2) {
            typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
            const u32x2u v = *reinterpret_cast<const u32x2u*>(p);
            f = f32x4{__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u), __uint_as_float(v[1] << 16),
                      __uint_as_float(v[1] & 0xffff0000u)};
        } else {
            typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
            const f32x4u v = *reinterpret_cast<const f32x4u*>(p);
            f = f32x4{v[0], v[1], v[2], v[3]};
        }
        return f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (c + i < C) f[i] = Elem<T>::load(p[i]);
    return f;
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Buffer descriptor of `bytes` bytes from p (both wave-uniform).  A lane whose offset lies outside reads zeros: that takes care of
// rows past the end, of the tail of a row and of steps that do not exist, without a branch around any copy.
__device__ __forceinline__ u32x4 f8_buffer(const unsigned char* p, unsigned bytes) {
    const uintptr_t b = (uintptr_t)p;
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b),
                 (unsigned)__builtin_amdgcn_readfirstlane((int)((b >> 32) & 0xffffu)),
                 (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
constexpr unsigned F8_OUTSIDE = 0xc0000000u;      // buffers are smaller than 2^31 bytes; what is added to this stays outside

// the same for the compiler's own buffer loads
__device__ __forceinline__ __amdgpu_buffer_rsrc_t f8_resource(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

// LDS-DMA through a buffer descriptor: 16 (4) bytes per lane to lds_wave_base + 16 (4) * lane; see glds16 for M0
__device__ __forceinline__ void buf_lds16(const u32x4& buf, unsigned voff, unsigned soff, unsigned lds_wave_base) {
    asm volatile(
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, %2 offen lds"
        :
        : "v"(voff), "s"(buf), "s"(soff), "s"(lds_wave_base)
        : "memory", "m0");
}
__device__ __forceinline__ void buf_lds4(const u32x4& buf, unsigned voff, unsigned soff, unsigned lds_wave_base) {
    asm volatile(
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dword %0, %1, %2 offen lds"
        :
        : "v"(voff), "s"(buf), "s"(soff), "s"(lds_wave_base)
        : "memory", "m0");
}

// Compute units of the current device (looked up once per device).
inline int f8_cus() {
    static int known[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (!known[dev]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
        known[dev] = n;
    }
    return known[dev];
}

}  // namespace mad
