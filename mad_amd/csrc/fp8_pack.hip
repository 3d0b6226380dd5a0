// Packing to and from the 8-bit block format (fp8.h): activations, the GroupNorm application that stores or restores
// its input as an 8-bit checkpoint on the way, and weights.
//
// All of it is bound by HBM: pack reads 2 (bf16) or 4 bytes per element and writes one, and so on.  A block of 128
// channels is the work of 16 lanes with eight elements each, so a block's maximum is a reduction over one row of lanes
// (four DPP steps), a wave covers four blocks and every access is a whole 16 (bytes: 8) per lane.  Measured in bf16: 65536 x 1152
// packed in 39.4 us and restored in 34.0 (229 MB: 5.8 and 6.7 TB/s), 32 x 128 x 128 x 256 normalised with its input saved in 120 us
// and restored in 101 (675 MB: 5.6 and 6.7 TB/s).
#include "fp8.h"

namespace mad {

// Streaming stores: what these passes write is larger than the caches that a following kernel could find it in, and kept there it
// displaces the input (restore of 32 x 128 x 128 x 256: 139 us with ordinary stores, 101 with these).
template <typename T> __device__ __forceinline__ void stream8_tail(T* p, int c, int C, const float* f) {
    if (c + 8 > C) { store8_tail<T>(p, c, C, f); return; }
    if constexpr (sizeof(T) == 2) {
        Vec16<bf16_t> t; t.pack(f); t.store_nt((bf16_t*)p);
    } else {
        Vec16<float> t; t.pack(f); t.store_nt((float*)p); t.pack(f + 4); t.store_nt((float*)p + 4);
    }
}
__device__ __forceinline__ void stream_q(unsigned char* p, const uint2& v) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    __builtin_nontemporal_store(u32x2{v.x, v.y}, reinterpret_cast<u32x2*>(p));
}

// The scale byte of block k of a row; the last block's lanes also write the padding behind it.
__device__ __forceinline__ void write_scale(unsigned char* row, unsigned s, int k, int kb, int sp, int l) {
    if (l < (k == kb - 1 ? sp - k : 1)) row[k + l] = (unsigned char)(l ? 127u : s);
}

// x (rows, C) -> q, scale.  One block per row of 16 lanes; a workgroup strides over the blocks.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void pack_fp8_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                                                       unsigned char* __restrict__ scale, long rows, int C) {
    const int kb = f8_blocks(C), pitch = f8_pitch(C), sp = f8_scale_pitch(C);
    const int l = threadIdx.x & 15;
    const long stride = (long)gridDim.x * 16;
    long b = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const long total = rows * kb;
    const long srow = stride / kb;
    const int scol = (int)(stride - srow * kb);
    long row = b / kb;
    int k = (int)(b - row * kb);
    for (; b < total; b += stride) {
        const int c = k * F8_BLOCK + 8 * l;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.0f;
        if (c < C) load8_tail<T>(x + row * C + c, c, C, f);
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { const unsigned u = f8_mag(f[i]); m = u > m ? u : m; }
        const unsigned s = f8_scale_byte<FMT>(row16_umax(m));
        const float inv = f8_inv_scale(s);
        if (c < pitch) {
            uint2 o;
            o.x = f8_cvt4<FMT>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
            o.y = f8_cvt4<FMT>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
            *reinterpret_cast<uint2*>(q + row * pitch + c) = o;
        }
        write_scale(scale + row * sp, s, k, kb, sp, l);
        row += srow; k += scol;
        if (k >= kb) { k -= kb; ++row; }
    }
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void unpack_fp8_kernel(const unsigned char* __restrict__ q,
                                                         const unsigned char* __restrict__ scale, T* __restrict__ x,
                                                         long rows, int C) {
    const int kb = f8_blocks(C), pitch = f8_pitch(C), sp = f8_scale_pitch(C);
    const int l = threadIdx.x & 15;
    const long stride = (long)gridDim.x * 16;
    const long total = rows * kb;
    const long srow = stride / kb;
    const int scol = (int)(stride - srow * kb);
    long b = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool whole = C * sizeof(T) % 16 == 0 && ((uintptr_t)x & 15) == 0;    // every piece of a row is aligned
    long row = b / kb;
    int k = (int)(b - row * kb);
    for (; b < total; b += stride) {
        const int c = k * F8_BLOCK + 8 * l;
        if (c < C) {
            const uint2 v = *reinterpret_cast<const uint2*>(q + row * pitch + c);
            const float s = f8_scale(scale[row * sp + k]);
            float f[8];
            f8_values4<FMT>(v.x, s, f);
            f8_values4<FMT>(v.y, s, f + 4);
            if (whole) stream8_tail<T>(x + row * C + c, c, C, f); else store8_tail<T>(x + row * C + c, c, C, f);
        }
        row += srow; k += scol;
        if (k >= kb) { k -= kb; ++row; }
    }
}

// y = drop(act(x*a + d)) as gn_apply_kernel computes it, and x as an 8-bit checkpoint (SAVE) or restored from one
// (!SAVE: x is written).  grid (pixel shares, B); a row of 16 lanes keeps its 128 channels, and their (a, d) in
// registers, over the pixels it walks.
template <typename T, bool SAVE>
__global__ __launch_bounds__(256) void gn_fp8_kernel(T* __restrict__ x, const float* __restrict__ coef, T* __restrict__ y,
                                                     unsigned char* __restrict__ q, unsigned char* __restrict__ scale,
                                                     int HW, int C, int act, DropMask dm) {
    const int kb = f8_blocks(C), pitch = f8_pitch(C), sp = f8_scale_pitch(C);
    const int l = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int b = blockIdx.y;
    // unsigned: a share that starts or ends behind the last pixel of the largest image (2^31 - 1 of them) does not fit an int
    const unsigned n = HW, per = (n + gridDim.x - 1) / gridDim.x;
    const unsigned p0 = blockIdx.x * per;
    const int pixels = p0 >= n ? 0 : n - p0 < per ? n - p0 : per;
    const size_t first = (size_t)b * n + p0;
    const int step = kb >= 16 ? 1 : 16 / kb;                  // pixels a workgroup covers per sweep
    for (int kbase = 0; kbase < kb; kbase += 16) {
        const int k = kbase + (kb >= 16 ? grp : grp % kb);
        const int row0 = kb >= 16 ? 0 : grp / kb;
        if (k >= kb || row0 >= step) continue;
        const int c = k * F8_BLOCK + 8 * l;
        float a[8], d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = d[i] = 0.0f;
        if (c < C) {
            const float* cf = coef + ((size_t)b * C + c) * 2;
            const int n = C - c < 8 ? C - c : 8;               // 4 (fp32) or 8
#pragma unroll
            for (int i = 0; i < 8; i += 2)
                if (i < n) {
                    const float4 v = *reinterpret_cast<const float4*>(cf + 2 * i);
                    a[i] = v.x; d[i] = v.y; a[i + 1] = v.z; d[i + 1] = v.w;
                }
        }
        for (int p = row0; p < pixels; p += step) {
            const size_t row = first + p;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = 0.0f;
            if (SAVE) {
                if (c < C) load8_tail<T>(x + row * C + c, c, C, f);
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) { const unsigned u = f8_mag(f[i]); m = u > m ? u : m; }
                const unsigned s = f8_scale_byte<F8_E4M3>(row16_umax(m));
                const float inv = f8_inv_scale(s);
                if (c < pitch) {
                    uint2 o;
                    o.x = f8_cvt4<F8_E4M3>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
                    o.y = f8_cvt4<F8_E4M3>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
                    stream_q(q + row * pitch + c, o);
                }
                write_scale(scale + row * sp, s, k, kb, sp, l);
            } else if (c < C) {
                const uint2 v = *reinterpret_cast<const uint2*>(q + row * pitch + c);
                const float s = f8_scale(scale[row * sp + k]);
                f8_values4<F8_E4M3>(v.x, s, f);
                f8_values4<F8_E4M3>(v.y, s, f + 4);
                stream8_tail<T>(x + row * C + c, c, C, f);
                // the activation is that of the restored tensor as it is stored
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = Elem<T>::load(Elem<T>::store(f[i]));
            }
            if (c >= C) continue;
            float r[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = fmaf(f[i], a[i], d[i]);
                r[i] = act ? silu_f(t) : t;
            }
            if (dm.thr) {                                     // the linear index of the element in y, as in gn_apply_kernel
                const unsigned long long e0 = (unsigned long long)row * C + c;
                float keep[4];
#pragma unroll
                for (int h = 0; h < 8; h += 4) {
                    drop_factors<4>(dm, e0 + h, keep);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[h + i] *= keep[i];
                }
            }
            stream8_tail<T>(y + row * C + c, c, C, r);
        }
    }
}

// Eight rows of eight bytes as their transpose: two rounds of v_perm on each 4 x 4 quarter.
__device__ __forceinline__ void transpose8x8(const uint2* in, uint2* out) {
    auto quarter = [](unsigned a, unsigned b, unsigned c, unsigned d, unsigned* o) {
        const unsigned ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);   // a0 b0 a1 b1
        const unsigned cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
        o[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u); o[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
        o[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u); o[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
    };
    unsigned t[4][4];
    quarter(in[0].x, in[1].x, in[2].x, in[3].x, t[0]);
    quarter(in[4].x, in[5].x, in[6].x, in[7].x, t[1]);
    quarter(in[0].y, in[1].y, in[2].y, in[3].y, t[2]);
    quarter(in[4].y, in[5].y, in[6].y, in[7].y, t[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) { out[i] = uint2{t[0][i], t[1][i]}; out[4 + i] = uint2{t[2][i], t[3][i]}; }
}

// One 128 x 128 block of a weight (N, K) per workgroup, 8 x 8 of it per thread: amax, the bytes as they lie, and transposed
// in registers and through LDS (8 bytes n of row k as piece n / 8 ^ k / 8).  4096 x 4096 from fp32, both copies: 19.2 us (with single
// bytes written to LDS 25.9), 100 MB at 5.2 TB/s; 137 x 200 4.6 (7.3).
template <typename T>
__global__ __launch_bounds__(256) void pack_weight_fp8_kernel(const T* __restrict__ w, int N, int K,
                                                              unsigned char* __restrict__ q, unsigned char* __restrict__ scale,
                                                              unsigned char* __restrict__ qt, unsigned char* __restrict__ scale_t) {
    __shared__ unsigned red[4];
    __shared__ __attribute__((aligned(16))) unsigned char tile[128 * 128];
    const int kbs = f8_scale_pitch(K), nbs = f8_scale_pitch(N);
    const int nb = blockIdx.x / kbs, kb = blockIdx.x - nb * kbs;
    const int nblocks = f8_blocks(N), kblocks = f8_blocks(K);
    const int tid = threadIdx.x, l = tid & 15, r = tid >> 4;
    if (nb >= nblocks || kb >= kblocks) {                     // padding of the scale rows
        if (tid == 0) {
            if (nb < nblocks) scale[(size_t)nb * kbs + kb] = 127;
            if (kb < kblocks && scale_t) scale_t[(size_t)kb * nbs + nb] = 127;
        }
        return;
    }
    const int n0 = nb * F8_BLOCK + 8 * r, c = kb * F8_BLOCK + 8 * l;
    float f[8][8];
    if ((nb + 1) * F8_BLOCK <= N && (kb + 1) * F8_BLOCK <= K) {
#pragma unroll
        for (int j = 0; j < 8; ++j) load8<T>(w + (size_t)(n0 + j) * K + c, f[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[j][i] = 0.0f;
            if (n0 + j < N && c < K) load8_tail<T>(w + (size_t)(n0 + j) * K + c, c, K, f[j]);
        }
    }
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) { const unsigned u = f8_mag(f[j][i]); m = u > m ? u : m; }
#pragma unroll
    for (int o = 32; o; o >>= 1) { const unsigned u = __shfl_xor(m, o); m = u > m ? u : m; }
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) m = red[i] > m ? red[i] : m;
    const unsigned s = f8_scale_byte<F8_E4M3>(m);
    const float inv = f8_inv_scale(s);
    const int kpitch = f8_pitch(K), npitch = f8_pitch(N);
    uint2 o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        o[j].x = f8_cvt4<F8_E4M3>(f[j][0] * inv, f[j][1] * inv, f[j][2] * inv, f[j][3] * inv);
        o[j].y = f8_cvt4<F8_E4M3>(f[j][4] * inv, f[j][5] * inv, f[j][6] * inv, f[j][7] * inv);
        if (n0 + j < N && c < kpitch) *reinterpret_cast<uint2*>(q + (size_t)(n0 + j) * kpitch + c) = o[j];
    }
    if (tid == 0) {
        scale[(size_t)nb * kbs + kb] = (unsigned char)s;
        if (qt) scale_t[(size_t)kb * nbs + nb] = (unsigned char)s;
    }
    if (!qt) return;
    uint2 ot[8];
    transpose8x8(o, ot);
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint2*>(tile + (8 * l + i) * 128 + ((r ^ l) << 3)) = ot[i];
    __syncthreads();
    const int n = nb * F8_BLOCK + 8 * l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int row = r + 16 * j, k = kb * F8_BLOCK + row;
        if (k < K && n < npitch)
            *reinterpret_cast<uint2*>(qt + (size_t)k * npitch + n) = *reinterpret_cast<const uint2*>(tile + row * 128 + ((l ^ (row >> 3)) << 3));
    }
}

// workgroups of 16 blocks each: enough that none walks many blocks (65536 x 1152 in bf16, us: pack 42.4 / 40.8 / 39.5 with at most 2048
// / 4096 / 8192, unpack 38.3 / 36.0 / 34.0 with 2048 / 4096 / 16384)
static int pack_grid(long blocks, long most) {
    const long g = (blocks + 15) / 16;
    return (int)(g < most ? (g > 0 ? g : 1) : most);
}

}  // namespace mad

using namespace mad;

static bool dtype_ok(int d) { return d == MAD_BF16 || d == MAD_F32; }

extern "C" int mad_pack_fp8(const void* x, int dtype, int fmt, long rows, int C, void* q, void* scale, void* stream) {
    MAD_REQUIRE(dtype_ok(dtype), "mad_pack_fp8: bad dtype %d", dtype);
    MAD_REQUIRE(fmt == MAD_E4M3 || fmt == MAD_E5M2, "mad_pack_fp8: bad 8-bit type %d", fmt);
    MAD_REQUIRE(rows >= 0 && C > 0 && C <= MAD_FP8_MAX_WIDTH, "mad_pack_fp8: bad shape %ld x %d", rows, C);
    if (rows == 0) return 0;
    MAD_REQUIRE(x && q && scale, "mad_pack_fp8: null pointer");
    MAD_REQUIRE(f8_aligned(q, scale), "mad_pack_fp8: q must be 16-byte, scale 4-byte aligned");
    const int grid = pack_grid(rows * f8_blocks(C), 8192);
#define LAUNCH(T, F)                                                                                                 \
    hipLaunchKernelGGL((pack_fp8_kernel<T, F>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const T*)x,            \
                       (unsigned char*)q, (unsigned char*)scale, rows, C)
    if (dtype == MAD_BF16) { if (fmt == MAD_E4M3) LAUNCH(bf16_t, F8_E4M3); else LAUNCH(bf16_t, F8_E5M2); }
    else { if (fmt == MAD_E4M3) LAUNCH(float, F8_E4M3); else LAUNCH(float, F8_E5M2); }
#undef LAUNCH
    return check_launch("mad_pack_fp8");
}

extern "C" int mad_unpack_fp8(const void* q, const void* scale, int fmt, long rows, int C, void* x, int dtype, void* stream) {
    MAD_REQUIRE(dtype_ok(dtype), "mad_unpack_fp8: bad dtype %d", dtype);
    MAD_REQUIRE(fmt == MAD_E4M3 || fmt == MAD_E5M2, "mad_unpack_fp8: bad 8-bit type %d", fmt);
    MAD_REQUIRE(rows >= 0 && C > 0 && C <= MAD_FP8_MAX_WIDTH, "mad_unpack_fp8: bad shape %ld x %d", rows, C);
    if (rows == 0) return 0;
    MAD_REQUIRE(x && q && scale, "mad_unpack_fp8: null pointer");
    MAD_REQUIRE(f8_aligned(q, scale), "mad_unpack_fp8: q must be 16-byte, scale 4-byte aligned");
    const int grid = pack_grid(rows * f8_blocks(C), 16384);
#define LAUNCH(T, F)                                                                                                 \
    hipLaunchKernelGGL((unpack_fp8_kernel<T, F>), dim3(grid), dim3(256), 0, (hipStream_t)stream,                       \
                       (const unsigned char*)q, (const unsigned char*)scale, (T*)x, rows, C)
    if (dtype == MAD_BF16) { if (fmt == MAD_E4M3) LAUNCH(bf16_t, F8_E4M3); else LAUNCH(bf16_t, F8_E5M2); }
    else { if (fmt == MAD_E4M3) LAUNCH(float, F8_E4M3); else LAUNCH(float, F8_E5M2); }
#undef LAUNCH
    return check_launch("mad_unpack_fp8");
}

template <bool SAVE>
static int gn_fp8(const char* what, void* x, const float* coef, void* y, void* q, void* scale, int dtype, int B, int HW, int C,
                  int act, unsigned long long seed, float p, void* stream) {
    MAD_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", what, dtype);
    const int VEC = dtype == MAD_BF16 ? 8 : 4;
    MAD_REQUIRE(C > 0 && C % VEC == 0 && C <= MAD_FP8_MAX_WIDTH, "%s: channels must be a multiple of %d (C=%d)", what, VEC, C);
    MAD_REQUIRE(B >= 0 && B <= 65535 && HW >= 0, "%s: bad shape B=%d HW=%d", what, B, HW);
    MAD_REQUIRE(p >= 0.0f && p < 1.0f, "%s: p=%f out of [0,1)", what, (double)p);
    if (B == 0 || HW == 0) return 0;
    MAD_REQUIRE(x && coef && y && q && scale, "%s: null pointer", what);
    MAD_REQUIRE(f8_aligned(q, scale), "%s: q must be 16-byte, scale 4-byte aligned", what);
    MAD_REQUIRE(!(((uintptr_t)x | (uintptr_t)y | (uintptr_t)coef) & 15), "%s: x, y and coef must be 16-byte aligned", what);
    // pixel shares: eight sweeps of pixels to a workgroup, or as few as keep 4096 workgroups (32 x 128 x 128 x 256, save / restore, us:
    // 134 / 108 with 2048 workgroups, 120 / 101 with 8192; 32 x 64 x 64 x 256 29 / 28 with 4096, 34 / 29 with 8192)
    const int kb = f8_blocks(C), step = kb >= 16 ? 1 : 16 / kb;
    const long sweeps = (long)B * (((long)HW + step - 1) / step);
    int shares = (int)(((sweeps / 8 > 4096 ? sweeps / 8 : 4096) + B - 1) / B);
    const int most = HW / step + (HW % step != 0);
    if (shares > most) shares = most;
    if (shares > 1 << 22) shares = 1 << 22;                                 // a launch counts fewer than 2^32 threads
    const DropMask dm = make_drop_mask(seed, p);
    if (dtype == MAD_BF16)
        hipLaunchKernelGGL((gn_fp8_kernel<bf16_t, SAVE>), dim3(shares, B), dim3(256), 0, (hipStream_t)stream, (bf16_t*)x, coef,
                           (bf16_t*)y, (unsigned char*)q, (unsigned char*)scale, HW, C, act, dm);
    else
        hipLaunchKernelGGL((gn_fp8_kernel<float, SAVE>), dim3(shares, B), dim3(256), 0, (hipStream_t)stream, (float*)x, coef,
                           (float*)y, (unsigned char*)q, (unsigned char*)scale, HW, C, act, dm);
    return check_launch(what);
}

extern "C" int mad_gn_apply_save_fp8(const void* x, const float* coef, void* y, void* q, void* scale, int dtype, int B, int HW,
                                     int C, int act, unsigned long long seed, float p, void* stream) {
    return gn_fp8<true>("mad_gn_apply_save_fp8", const_cast<void*>(x), coef, y, q, scale, dtype, B, HW, C, act, seed, p, stream);
}

extern "C" int mad_gn_apply_restore_fp8(const void* q, const void* scale, const float* coef, void* x, void* y, int dtype, int B,
                                        int HW, int C, int act, unsigned long long seed, float p, void* stream) {
    return gn_fp8<false>("mad_gn_apply_restore_fp8", x, coef, y, const_cast<void*>(q), const_cast<void*>(scale), dtype, B, HW, C,
                         act, seed, p, stream);
}

extern "C" int mad_pack_weight_fp8(const void* w, int dtype, int N, int K, void* q, void* scale, void* qt, void* scale_t,
                                   void* stream) {
    MAD_REQUIRE(dtype_ok(dtype), "mad_pack_weight_fp8: bad dtype %d", dtype);
    MAD_REQUIRE(N > 0 && K > 0 && N <= MAD_FP8_MAX_WIDTH && K <= MAD_FP8_MAX_WIDTH, "mad_pack_weight_fp8: bad shape %d x %d", N, K);
    MAD_REQUIRE(w && q && scale && (!qt == !scale_t), "mad_pack_weight_fp8: null pointer");
    MAD_REQUIRE(f8_aligned(q, scale) && f8_aligned(qt, scale_t), "mad_pack_weight_fp8: bytes must be 16-byte, scales 4-byte aligned");
    // whole groups of four blocks in both directions: their padding is written too
    const dim3 grid((unsigned)f8_scale_pitch(N) * (unsigned)f8_scale_pitch(K));
    if (dtype == MAD_BF16)
        hipLaunchKernelGGL(pack_weight_fp8_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16_t*)w, N, K,
                           (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t);
    else
        hipLaunchKernelGGL(pack_weight_fp8_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)w, N, K,
                           (unsigned char*)q, (unsigned char*)scale, (unsigned char*)qt, (unsigned char*)scale_t);
    return check_launch("mad_pack_weight_fp8");
}
