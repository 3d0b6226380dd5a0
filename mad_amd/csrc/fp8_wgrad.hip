// Weight gradient of a layer whose input was kept in 8 bits (fp8.h):
//
//   dw[n][k] (+)= sum_m dy[m][n] * x[m][k]      db[n] (+)= sum_m dy[m][n]
//
// The scale of x changes along the reduction (one per row m), so the product cannot run on 8-bit operands; but bf16 holds
// every restored value exactly, so x is widened on its way into LDS and the product runs on v_mfma_f32_16x16x32_bf16 without a
// further rounding.  dy is bf16, or fp32 cut into three bf16 terms whose sum is dy to 24 bits (x is exact, so three
// products give fp32 accuracy).  Both operands are stored with the reduction index slow and read with the transposing LDS
// read (ds_read_b64_tr_b16: a row of 16 lanes fetches 4 rows m x 16 columns, lane i receives column i).
// Shares of the rows write partial sums that a second kernel adds in share order: the result does not depend on timing.
#include "fp8.h"

namespace mad {

struct F8WgradArgs {
    const void* dy; const unsigned char* x; const unsigned char* xs;
    float* dw; float* db;                      // destinations, or partial slabs when splits > 1
    long M, per;                               // rows, rows per share (a multiple of 32)
    int N, K, ntiles, ktiles, splits, acc_w, acc_b;
};

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

__device__ __forceinline__ bf16x8 tr_pair(const unsigned char* lo, const unsigned char* hi) {
    const bf16x4 l = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)lo);
    const bf16x4 h = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)hi);
    return bf16x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
}

__device__ __forceinline__ uint4 pack8_bf16(const float* f) {
    uint4 o;
    unsigned* w = &o.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (unsigned)f32_to_bf16(f[2 * i]) | ((unsigned)f32_to_bf16(f[2 * i + 1]) << 16);
    return o;
}

// T: type of dy; FMT: 8-bit type of x.  A workgroup owns 128 (n) x 128 (k) of dw and a share of the rows; four waves 2 x 2
// of 64 x 64.  LDS tiles [32 rows m][128 columns] bf16; the 16-byte chunk c of row m lies at c ^ ((m & 3) << 2), so the four
// rows a transposing read touches are in different banks.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void wgrad_fp8_kernel(F8WgradArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;               // bf16 terms of dy
    constexpr int TILE = 32 * 256;
    __shared__ __attribute__((aligned(16))) unsigned char smem[(NP + 1) * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave >> 1, wk = wave & 1;
    const int tiles = a.ntiles * a.ktiles;
    const int split = blockIdx.x / tiles, t = blockIdx.x - split * tiles;
    const int nt = t / a.ktiles, kt = t - nt * a.ktiles;
    const int n0 = nt * 128, k0 = kt * 128;
    const long m_begin = (long)split * a.per, m_end = m_begin + a.per < a.M ? m_begin + a.per : a.M;
    const int xp = f8_pitch(a.K), sp = f8_scale_pitch(a.K);
    const T* dy = (const T*)a.dy;

    f32x4 acc[4][4], accb[4];                                 // [k fragment][n fragment]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        accb[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const bool with_bias = a.db && kt == 0 && wk == 0;        // column sums: the gradient of an input column of ones
    const __bf16 one = (__bf16)1.0f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};

    const int lr = tid >> 4, lc = tid & 15;                   // loader: row within 16, 8-column piece
    const int g = lane >> 4, q = (lane >> 2) & 3, pp = lane & 3;
    auto frag = [&](const unsigned char* tile, int col) {     // 16 columns from col, all 32 rows
        const int chunk = (col >> 3) + (pp >> 1);
        const int off = ((chunk ^ (q << 2)) << 4) + (pp & 1) * 8;
        return tr_pair(tile + (4 * g + q) * 256 + off, tile + (16 + 4 * g + q) * 256 + off);
    };

    for (long m = m_begin; m < m_end; m += 32) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = 16 * h + lr;
            const long mr = m + row;
            const bool live = mr < m_end;
            unsigned char* dst = smem + row * 256 + ((lc ^ ((row & 3) << 2)) << 4);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = 0.0f;
            const int n = n0 + 8 * lc, c = k0 + 8 * lc;
            if (live && n < a.N) load8_tail<T>(dy + (size_t)mr * a.N + n, n, a.N, f);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                *reinterpret_cast<uint4*>(dst + p * TILE) = pack8_bf16(f);
                if (p + 1 < NP) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {              // what the terms so far leave (nothing of an infinity or NaN)
                        const float hi = bf16_to_f32(f32_to_bf16(f[e]));
                        f[e] = f8_mag(hi) || hi == 0.0f ? f[e] - hi : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = 0.0f;
            if (live && c < xp) {
                const uint2 v = *reinterpret_cast<const uint2*>(a.x + (size_t)mr * xp + c);
                const float s = f8_scale(a.xs[(size_t)mr * sp + kt]);
                f8_values4<FMT>(v.x, s, f);
                f8_values4<FMT>(v.y, s, f + 4);
            }
            *reinterpret_cast<uint4*>(dst + NP * TILE) = pack8_bf16(f);
        }
        __syncthreads();
        bf16x8 xf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xf[i] = frag(smem + NP * TILE, wk * 64 + 16 * i);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x8 d = frag(smem + p * TILE, wn * 64 + 16 * j);
                if (with_bias) accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, d, accb[j], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], d, acc[i][j], 0, 0, 0);
            }
    }

    // a lane holds four consecutive k of one n
    const bool direct = a.splits == 1;
    float* dw = a.dw + (direct ? 0 : (size_t)split * a.N * a.K);
    const int r = lane & 15;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = n0 + wn * 64 + 16 * j + r;
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + wk * 64 + 16 * i + 4 * g;
            float* p = dw + (size_t)n * a.K + k;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k + e < a.K) p[e] = (direct && a.acc_w ? p[e] : 0.0f) + acc[i][j][e];
        }
        if (with_bias && g == 0) {
            float* p = a.db + (direct ? 0 : (size_t)split * a.N) + n;
            *p = (direct && a.acc_b ? *p : 0.0f) + accb[j][0];
        }
    }
}

// dst[i] (+)= sum of the shares' partial sums, in share order
__global__ __launch_bounds__(256) void wgrad_fp8_join_kernel(const float* __restrict__ part, float* __restrict__ dst, size_t n,
                                                             int splits, int accumulate) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int z = 0; z < splits; ++z) s += part[(size_t)z * n + i];
        dst[i] = accumulate ? dst[i] + s : s;
    }
}

// Shares of the rows: enough workgroups to fill the chip, at least 256 rows each.
static int wgrad_splits(long rows, int N, int K) {
    const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128);
    long s = (512 + tiles - 1) / tiles;
    const long most = (rows + 255) / 256;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}

}  // namespace mad

using namespace mad;

static bool wgrad_shape_ok(long rows, int N, int K) {
    return rows >= 0 && N > 0 && N <= MAD_FP8_MAX_WIDTH && K > 0 && K <= MAD_FP8_MAX_WIDTH;
}

extern "C" size_t mad_linear_fp8_wgrad_workspace(long rows, int N, int K) {
    if (!wgrad_shape_ok(rows, N, K)) return 0;
    const int s = wgrad_splits(rows, N, K);
    return s > 1 ? (size_t)s * ((size_t)N * K + N) * sizeof(float) : 0;
}

extern "C" int mad_linear_fp8_wgrad(const void* dy, int dtype, const void* x, int x_type, const void* x_scale, float* dw, float* db,
                                    void* workspace, size_t workspace_bytes, long rows, int N, int K, int accumulate,
                                    int bias_accumulate, void* stream) {
    MAD_REQUIRE(dtype == MAD_BF16 || dtype == MAD_F32, "mad_linear_fp8_wgrad: bad dtype %d", dtype);
    MAD_REQUIRE(x_type == MAD_E4M3 || x_type == MAD_E5M2, "mad_linear_fp8_wgrad: x is of type %d, not an 8-bit one", x_type);
    MAD_REQUIRE(wgrad_shape_ok(rows, N, K), "mad_linear_fp8_wgrad: bad shape rows=%ld N=%d K=%d", rows, N, K);
    MAD_REQUIRE(dw && (rows == 0 || (dy && x && x_scale)), "mad_linear_fp8_wgrad: null pointer");
    MAD_REQUIRE(f8_aligned(x, x_scale), "mad_linear_fp8_wgrad: x must be 16-byte, its scales 4-byte aligned");
    F8WgradArgs a;
    a.dy = dy; a.x = (const unsigned char*)x; a.xs = (const unsigned char*)x_scale;
    a.M = rows; a.N = N; a.K = K;
    a.splits = wgrad_splits(rows, N, K);
    const size_t need = mad_linear_fp8_wgrad_workspace(rows, N, K);
    MAD_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "mad_linear_fp8_wgrad: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    a.per = ((rows + a.splits - 1) / a.splits + 31) / 32 * 32;
    a.ntiles = (N + 127) / 128; a.ktiles = (K + 127) / 128;
    a.acc_w = accumulate; a.acc_b = bias_accumulate;
    const size_t nk = (size_t)N * K;
    float* part_b = a.splits > 1 ? (float*)workspace + (size_t)a.splits * nk : nullptr;
    a.dw = a.splits > 1 ? (float*)workspace : dw;
    a.db = db ? (a.splits > 1 ? part_b : db) : nullptr;
    const long wgs = (long)a.ntiles * a.ktiles * a.splits;
    MAD_REQUIRE(wgs <= 0x7fffffffL, "mad_linear_fp8_wgrad: N=%d K=%d need more workgroups than a launch holds", N, K);
    hipStream_t s = (hipStream_t)stream;
#define LAUNCH(T, F) hipLaunchKernelGGL((wgrad_fp8_kernel<T, F>), dim3((unsigned)wgs), dim3(256), 0, s, a)
    if (dtype == MAD_BF16) { if (x_type == MAD_E4M3) LAUNCH(bf16_t, F8_E4M3); else LAUNCH(bf16_t, F8_E5M2); }
    else { if (x_type == MAD_E4M3) LAUNCH(float, F8_E4M3); else LAUNCH(float, F8_E5M2); }
#undef LAUNCH
    if (int rc = check_launch("mad_linear_fp8_wgrad")) return rc;
    if (a.splits > 1) {
        const size_t blocks = (nk + 255) / 256;
        hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s,
                           (const float*)workspace, dw, nk, a.splits, accumulate);
        if (db)
            hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, (const float*)part_b, db,
                               (size_t)N, a.splits, bias_accumulate);
        return check_launch("mad_linear_fp8_wgrad");
    }
    return 0;
}
