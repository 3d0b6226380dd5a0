// Matrix products of 8-bit operands in the block format of fp8.h:
//
//   y[m][n] = bias[n] + sum_k x[m][k] * w[n][k] (+ residual[m][n])
//
// with x (rows, K) one scale per row and 128 columns and w (N, K) one scale per 128 x 128 block.  One
// v_mfma_f32_16x16x128_f8f6f4 takes 16 rows of each operand over one whole block, and applies both scales itself.  Which
// 32 of the 128 columns a lane holds does not matter as long as both operands agree, since they share their scales.
//
// Accuracy.  The 8-bit matrix instructions add the products of eight consecutive columns on one exponent: measured, a product
// loses what lies below 2^-13 of the largest of its eight (cut toward zero), and only the eights are added in full fp32.
// That is 1.6e-5 of the result (2-norm, normal operands), far below the 2^-9 of a bf16 result, so y in bf16 takes them.
// y in fp32 widens the bytes to bf16 (exact) and takes v_mfma_f32_16x16x32_bf16, whose sums are fp32 throughout, block by
// block; the block's sum is then scaled and added.  Half the rate or less, 1e-7 of the result.
//
// The weights are the FIRST operand, so a lane's four results are four consecutive columns n of one row m.
#include "fp8.h"

namespace mad {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct F8LinArgs {
    const void* x; const unsigned char* xs;        // x as bytes with scales, or as bf16 / fp32 (xs null)
    const unsigned char* w; const unsigned char* ws;
    const float* bias; const void* residual; void* y;
    long M;
    int K, N, ntiles;
    int quads;                                     // rows of y are whole quads and every quad is aligned
};

// kinds of x
constexpr int X_E4M3 = 0, X_E5M2 = 1, X_BF16 = 2, X_F32 = 3;

__device__ __forceinline__ i32x8 pair16(const uint4& a, const uint4& b) {
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// Four consecutive columns n .. n+3 of row m: bias, residual, one rounding, store.
template <typename TO>
__device__ __forceinline__ void store_quad(const F8LinArgs& a, long m, int n, f32x4 v) {
    if (m >= a.M || n >= a.N) return;
    TO* y = (TO*)a.y + m * a.N + n;
    const TO* r = a.residual ? (const TO*)a.residual + m * a.N + n : nullptr;
    if (a.quads) {
        if (a.bias) v += *reinterpret_cast<const f32x4*>(a.bias + n);
        if constexpr (sizeof(TO) == 4) {
            if (r) v += *reinterpret_cast<const f32x4*>(r);
            *reinterpret_cast<f32x4*>(y) = v;
        } else {
            if (r) {
                const uint2 t = *reinterpret_cast<const uint2*>(r);
                v += f32x4{__uint_as_float(t.x << 16), __uint_as_float(t.x & 0xffff0000u), __uint_as_float(t.y << 16),
                           __uint_as_float(t.y & 0xffff0000u)};
            }
            uint2 o;
            o.x = (unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16);
            o.y = (unsigned)f32_to_bf16(v[2]) | ((unsigned)f32_to_bf16(v[3]) << 16);
            *reinterpret_cast<uint2*>(y) = o;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.N) {
            float s = v[e] + (a.bias ? a.bias[n + e] : 0.0f);
            if (r) s += Elem<TO>::load(r[e]);
            y[e] = Elem<TO>::store(s);
        }
}

// acc += one block of 128 columns, 32 of them in this lane: see "Accuracy" above.
template <int XF, bool EXACT>
__device__ __forceinline__ void block_product(f32x4& acc, const i32x8& w, const i32x8& x, int wscale, int xscale) {
    if constexpr (!EXACT) {
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, F8_E4M3, XF, 0, wscale, 0, xscale);
    } else {
        f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < 4; ++q)
            t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f8_bf16x8<F8_E4M3>(w[2 * q], w[2 * q + 1]), f8_bf16x8<XF>(x[2 * q], x[2 * q + 1]),
                                                        t, 0, 0, 0);
        // the lane's column of t is row lane & 15 of x, whose scale it holds
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __builtin_amdgcn_ldexpf(t[e], wscale + xscale - 254);
    }
}

// Direct form: operands from global memory straight into registers, (16 MF) x (16 NF) outputs per workgroup, its NW
// waves taking every NW-th block of the reduction; their sums are added in wave order through LDS.
template <int XK, typename TO, int MF, int NF, int NW>
__global__ __launch_bounds__(64 * NW) void linear_fp8_direct_kernel(F8LinArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 red[NW > 1 ? NW : 1][MF * NF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const long mt = blockIdx.x / a.ntiles;
    const int nt = (int)(blockIdx.x - mt * a.ntiles);
    const long m0 = mt * (16 * MF);
    const int n0 = nt * (16 * NF);
    const int kb = f8_blocks(a.K), wp = f8_pitch(a.K), sp = f8_scale_pitch(a.K);

    f32x4 acc[NF][MF];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int kt = wave; kt < kb; kt += NW) {
        const int c = kt * F8_BLOCK + 32 * g;
        i32x8 wf[NF], xf[MF];
        int wsc[NF], xsc[MF];
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            int n = n0 + 16 * j + r;
            n = n < a.N ? n : a.N - 1;                 // rows past the end repeat the last one: their results are not stored
            const unsigned char* p = a.w + (size_t)n * wp + c;
            uint4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
            if (c < wp) lo = *reinterpret_cast<const uint4*>(p);
            if (c + 16 < wp) hi = *reinterpret_cast<const uint4*>(p + 16);
            wf[j] = pair16(lo, hi);
            wsc[j] = a.ws[(size_t)(n / F8_BLOCK) * sp + kt];
        }
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            long m = m0 + 16 * i + r;
            m = m < a.M ? m : a.M - 1;
            if constexpr (XK < X_BF16) {
                const unsigned char* p = (const unsigned char*)a.x + (size_t)m * wp + c;
                uint4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
                if (c < wp) lo = *reinterpret_cast<const uint4*>(p);
                if (c + 16 < wp) hi = *reinterpret_cast<const uint4*>(p + 16);
                xf[i] = pair16(lo, hi);
                xsc[i] = a.xs[(size_t)m * sp + kt];
            } else {
                using T = typename std::conditional<XK == X_BF16, bf16_t, float>::type;
                const T* p = (const T*)a.x + (size_t)m * a.K + c;
                float f[32];
                unsigned u = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) load8_tail<T>(p + 8 * q, c + 8 * q, a.K, f + 8 * q);
#pragma unroll
                for (int e = 0; e < 32; ++e) { const unsigned t = f8_mag(f[e]); u = t > u ? t : u; }
                // the row's block: this lane's quarter and those of the lanes 16, 32 and 48 on
                unsigned t = __shfl_xor(u, 16); u = t > u ? t : u;
                t = __shfl_xor(u, 32); u = t > u ? t : u;
                const unsigned s = f8_scale_byte<F8_E4M3>(u);
                const float inv = f8_inv_scale(s);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    xf[i][q] = (int)f8_cvt4<F8_E4M3>(f[4 * q] * inv, f[4 * q + 1] * inv, f[4 * q + 2] * inv, f[4 * q + 3] * inv);
                xsc[i] = (int)s;
            }
        }
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i)
                block_product<XK == X_E5M2 ? F8_E5M2 : F8_E4M3, sizeof(TO) == 4>(acc[j][i], wf[j], xf[i], wsc[j], xsc[i]);
    }
    if constexpr (NW > 1) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i) red[wave][j * MF + i][lane] = acc[j][i];
        __syncthreads();
        for (int f = wave; f < MF * NF; f += NW) {
            f32x4 v = red[0][f][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) v += red[w][f][lane];
            store_quad<TO>(a, m0 + 16 * (f % MF) + r, n0 + 16 * (f / MF) + 4 * g, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i) store_quad<TO>(a, m0 + 16 * i + r, n0 + 16 * j + 4 * g, acc[j][i]);
    }
}

template <int XK, typename TO> static int launch_linear(F8LinArgs a, hipStream_t s) {
    constexpr int MF = 4, NF = 4, NW = 4;
    const long mtiles = (a.M + 16 * MF - 1) / (16 * MF);
    a.ntiles = (a.N + 16 * NF - 1) / (16 * NF);
    MAD_REQUIRE(mtiles * a.ntiles <= 0x7fffffffL, "mad_linear_fp8: %ld rows x %d columns need more workgroups than a launch holds",
                a.M, a.N);
    hipLaunchKernelGGL((linear_fp8_direct_kernel<XK, TO, MF, NF, NW>), dim3((unsigned)(mtiles * a.ntiles)), dim3(64 * NW), 0, s, a);
    return check_launch("mad_linear_fp8");
}

}  // namespace mad

using namespace mad;

extern "C" int mad_linear_fp8(const void* x, int x_type, const void* x_scale, const void* w, const void* w_scale,
                              const float* bias, const void* residual, void* y, int dtype, long rows, int K, int N,
                              void* stream) {
    MAD_REQUIRE(dtype == MAD_BF16 || dtype == MAD_F32, "mad_linear_fp8: bad dtype %d", dtype);
    MAD_REQUIRE(x_type == MAD_E4M3 || x_type == MAD_E5M2 || x_type == dtype,
                "mad_linear_fp8: x is of type %d: 8-bit, or the type of y (%d)", x_type, dtype);
    MAD_REQUIRE(rows >= 0 && K > 0 && K <= MAD_FP8_MAX_WIDTH && N > 0 && N <= MAD_FP8_MAX_WIDTH,
                "mad_linear_fp8: bad shape rows=%ld K=%d N=%d", rows, K, N);
    if (rows == 0) return 0;
    const bool packed = x_type == MAD_E4M3 || x_type == MAD_E5M2;
    MAD_REQUIRE(x && w && w_scale && y && (!packed || x_scale), "mad_linear_fp8: null pointer");
    MAD_REQUIRE(f8_aligned(w, w_scale) && (!packed || f8_aligned(x, x_scale)),
                "mad_linear_fp8: packed bytes must be 16-byte, scales 4-byte aligned");
    F8LinArgs a;
    a.x = x; a.xs = (const unsigned char*)x_scale; a.w = (const unsigned char*)w; a.ws = (const unsigned char*)w_scale;
    a.bias = bias; a.residual = residual; a.y = y; a.M = rows; a.K = K; a.N = N; a.ntiles = 0;
    const uintptr_t es = dtype == MAD_BF16 ? 2 : 4;
    a.quads = N % 4 == 0 && !((uintptr_t)bias & 15) && !(((uintptr_t)residual | (uintptr_t)y) & (4 * es - 1));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MAD_BF16) {
        if (x_type == MAD_E4M3) return launch_linear<X_E4M3, bf16_t>(a, s);
        if (x_type == MAD_E5M2) return launch_linear<X_E5M2, bf16_t>(a, s);
        return launch_linear<X_BF16, bf16_t>(a, s);
    }
    if (x_type == MAD_E4M3) return launch_linear<X_E4M3, float>(a, s);
    if (x_type == MAD_E5M2) return launch_linear<X_E5M2, float>(a, s);
    return launch_linear<X_F32, float>(a, s);
}
