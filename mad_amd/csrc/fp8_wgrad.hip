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
//
// db is the gradient of an input column of ones: one more product per fragment of dy.  A workgroup makes it for every
// ktiles-th step only (kt = step mod ktiles), so that no tile of dw has more work than another; the parts are joined.
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
    const bool with_bias = a.db && wk == 0;
    int turn = 0;                                             // step mod ktiles
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
        const bool mine = with_bias && turn == kt;
        turn = turn + 1 == a.ktiles ? 0 : turn + 1;
        bf16x8 xf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xf[i] = frag(smem + NP * TILE, wk * 64 + 16 * i);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x8 d = frag(smem + p * TILE, wn * 64 + 16 * j);
                if (mine) accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, d, accb[j], 0, 0, 0);
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
            float* p = a.db + ((size_t)split * a.ktiles + kt) * a.N + n;
            *p = (a.acc_b ? *p : 0.0f) + accb[j][0];
        }
    }
}

// Tiled form: dy in bf16 with rows of whole 16-byte pieces.  BN (n) x BK (k) of dw per workgroup of WN x WK waves, 64 rows m per
// step, two LDS stages.  dy comes by LDS-DMA; x is loaded into registers one step ahead and widened into LDS after the step's
// products, so that one barrier per step remains.  Columns past the end read what lies there, which only reaches results that
// are not stored; rows past the share are zeros (buffer loads outside their buffer).
template <int BN, int BK> struct F8Wg {
    static constexpr int ROWS = 64, DY = ROWS * BN * 2, STAGE = DY + ROWS * BK * 2, LDS = 2 * STAGE;
};

template <int FMT, int BN, int BK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) void wgrad_fp8_tile_kernel(F8WgradArgs a) {
    using L = F8Wg<BN, BK>;
    constexpr int NW = WN * WK, FN = BN / WN / 16, FK = BK / WK / 16;
    constexpr int DPW = BN / 8 / NW;                                      // dy copies per wave and step (4 rows x 128 columns each)
    constexpr int XPT = 64 * BK / 16 / (64 * NW);                         // 16-byte pieces of x per thread and step
    static_assert(BN % 128 == 0 && BK % 128 == 0 && BN % (8 * NW) == 0 && XPT * 16 * NW == BK, "tile");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / WK, wk = wave % WK;
    const int g = lane >> 4, q = (lane >> 2) & 3, pp = lane & 3;

    // an XCD takes a run of consecutive (share, tile): the tiles of a share read the same rows
    const int tiles = a.ntiles * a.ktiles, nwg = gridDim.x, id = blockIdx.x;
    const int q8 = nwg >> 3, r8 = nwg & 7, xcd = id & 7;
    const int logical = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (id >> 3);
    const int split = __builtin_amdgcn_readfirstlane(logical / tiles), t = logical - split * tiles;
    const int per = 8 * a.ktiles, grp = t / per, in = t - grp * per;
    const int gn = a.ntiles - 8 * grp < 8 ? a.ntiles - 8 * grp : 8, col = in / gn;
    const int kt = __builtin_amdgcn_readfirstlane(col), nt = __builtin_amdgcn_readfirstlane(8 * grp + in - col * gn);
    const int n0 = nt * BN, k0 = kt * BK;
    const long m_begin = (long)split * a.per, m_end = m_begin + a.per < a.M ? m_begin + a.per : a.M;
    const int steps = (int)((m_end - m_begin + L::ROWS - 1) / L::ROWS);
    const int xp = f8_pitch(a.K), sp = f8_scale_pitch(a.K), kb = f8_blocks(a.K);

    // where this lane's copies read: offsets inside the 64 rows of a step
    const int lr = lane >> 4;
    unsigned doff[DPW];
#pragma unroll
    for (int j = 0; j < DPW; ++j) {
        const int c = j * NW + wave;                                      // half c / 16, rows 4 (c % 16) ..
        doff[j] = (unsigned)((4 * (c & 15) + lr) * a.N * 2 + (n0 + (c >> 4) * 128) * 2 + (((lane & 15) ^ (lr << 2)) << 4));
    }
    unsigned xoff[XPT], soff[XPT];
    int xdst[XPT];
#pragma unroll
    for (int u = 0; u < XPT; ++u) {
        const int i = u * 64 * NW + tid, row = i / (BK / 16), piece = i % (BK / 16), half = piece >> 3;
        xoff[u] = (unsigned)(row * xp + k0 + 16 * piece);
        const int block = k0 / F8_BLOCK + half;
        soff[u] = (unsigned)(row * sp + (block < kb ? block : kb - 1));
        xdst[u] = L::DY + (half * L::ROWS + row) * 256 + (((2 * (piece & 7)) ^ ((row & 3) << 2)) << 4);
    }
    const unsigned lds0 = lds_addr(smem);
    uint4 xr[XPT];
    unsigned sr[XPT];
    auto fetch = [&](int s, int buf) {                                    // step s: dy into its stage, x into registers
        const long m = m_begin + (long)s * L::ROWS;
        const int rows = m_end - m < L::ROWS ? (int)(m_end - m) : L::ROWS;
        const u32x4 db = f8_buffer((const unsigned char*)a.dy + (size_t)m * a.N * 2, (unsigned)(rows * a.N * 2));
#pragma unroll
        for (int j = 0; j < DPW; ++j) buf_lds16(db, doff[j], 0, lds0 + buf * L::STAGE + (j * NW + wave) * 1024);
        const auto xrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (size_t)m * xp), 0, rows * xp, 0x00020000);
        const auto srs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.xs + (size_t)m * sp), 0, rows * sp, 0x00020000);
#pragma unroll
        for (int u = 0; u < XPT; ++u) {
            xr[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(xrs, (int)xoff[u], 0, 0));
            sr[u] = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(srs, (int)soff[u], 0, 0);
        }
    };
    auto widen = [&](int buf) {                                           // the fetched x into the stage
#pragma unroll
        for (int u = 0; u < XPT; ++u) {
            const float s = f8_scale(sr[u]);
            unsigned char* d = smem + buf * L::STAGE;
            *reinterpret_cast<bf16x8*>(d + xdst[u]) = f8_bf16x8<FMT>(xr[u].x, xr[u].y, s);
            *reinterpret_cast<bf16x8*>(d + (xdst[u] ^ 16)) = f8_bf16x8<FMT>(xr[u].z, xr[u].w, s);
        }
    };

    f32x4 acc[FK][FN], accb[FN];                              // [k fragment][n fragment]
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        accb[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < FK; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const __bf16 one = (__bf16)1.0f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};
    const bool with_bias = a.db && wk == 0;
    int turn = 0;

    // fragment of 16 columns: rows 4g + q and 16 rows on, 8 bytes at columns 4 pp
    const int frow = (4 * g + q) * 256 + (pp & 1) * 8;
    auto frag = [&](const unsigned char* tile, int c, int h) {
        const int chunk = ((c & 127) >> 3) + (pp >> 1);
        const unsigned char* p = tile + (c >> 7) * L::ROWS * 256 + h * 32 * 256 + frow + ((chunk ^ (q << 2)) << 4);
        return tr_pair(p, p + 16 * 256);
    };

    if (steps > 0) { fetch(0, 0); widen(0); }
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        dma_wait_all();
        __syncthreads();                   // step s is visible; every wave is done with the stage refilled below
        if (s + 1 < steps) fetch(s + 1, buf ^ 1);
        const bool mine = with_bias && turn == kt;
        turn = turn + 1 == a.ktiles ? 0 : turn + 1;
        const unsigned char* st = smem + buf * L::STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 xf[FK];
#pragma unroll
            for (int i = 0; i < FK; ++i) xf[i] = frag(st + L::DY, wk * (BK / WK) + 16 * i, h);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const bf16x8 d = frag(st, wn * (BN / WN) + 16 * j, h);
                if (mine) accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, d, accb[j], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < FK; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], d, acc[i][j], 0, 0, 0);
            }
        }
        if (s + 1 < steps) widen(buf ^ 1);
    }

    // a lane holds four consecutive k of one n
    const bool direct = a.splits == 1;
    float* dw = a.dw + (direct ? 0 : (size_t)split * a.N * a.K);
    const int r = lane & 15;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn * (BN / WN) + 16 * j + r;
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < FK; ++i) {
            const int k = k0 + wk * (BK / WK) + 16 * i + 4 * g;
            if (k >= a.K) continue;
            float* p = dw + (size_t)n * a.K + k;
            f32x4 v = acc[i][j];
            if (direct && a.acc_w) v += load4_tail<float>(p, k, a.K);
            store4_tail<float>(p, k, a.K, v);
        }
        if (with_bias && g == 0) {
            float* p = a.db + ((size_t)split * a.ktiles + kt) * a.N + n;
            *p = (a.acc_b ? *p : 0.0f) + accb[j][0];
        }
    }
}

// dst[i] (+)= sum of the parts' partial sums, in order
__global__ __launch_bounds__(256) void wgrad_fp8_join_kernel(const float* __restrict__ part, float* __restrict__ dst, size_t n,
                                                             int parts, int accumulate) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int z = 0; z < parts; ++z) s += part[(size_t)z * n + i];
        dst[i] = accumulate ? dst[i] + s : s;
    }
}

// How a gradient is cut: the form, its tiles and the shares of the rows.
struct F8WgradPlan { int tile, ntiles, ktiles, splits; long per; };

static F8WgradPlan wgrad_plan(long rows, int N, int K, bool tiled) {
    F8WgradPlan p;
    auto tiles = [&](int t) { return (long)((N + t - 1) / t) * ((K + t - 1) / t); };
    const int cus = f8_cus();
    p.tile = tiled && tiles(256) >= cus ? 256 : 128;
    p.ntiles = (N + p.tile - 1) / p.tile; p.ktiles = (K + p.tile - 1) / p.tile;
    long s = (2 * cus + tiles(p.tile) - 1) / tiles(p.tile);
    if (p.tile == 256) s = 1;
    const long most = (rows + 255) / 256;
    if (s > most) s = most;
    p.splits = (int)(s < 1 ? 1 : s);
    p.per = ((rows + p.splits - 1) / p.splits + 63) / 64 * 64;
    return p;
}

}  // namespace mad

using namespace mad;

static bool wgrad_shape_ok(long rows, int N, int K) {
    return rows >= 0 && N > 0 && N <= MAD_FP8_MAX_WIDTH && K > 0 && K <= MAD_FP8_MAX_WIDTH;
}

static size_t wgrad_workspace(const F8WgradPlan& p, int N, int K) {
    const size_t w = p.splits > 1 ? (size_t)p.splits * N * K : 0;
    const size_t b = (size_t)p.splits * p.ktiles > 1 ? (size_t)p.splits * p.ktiles * N : 0;
    return (w + b) * sizeof(float);
}

// the form with LDS-DMA of dy needs whole 16-byte pieces, and 64 rows within a buffer's 32-bit offsets
static bool wgrad_tiled(const void* dy, int dtype, int N) {
    return dtype == MAD_BF16 && N % 8 == 0 && !((uintptr_t)dy & 15);
}

extern "C" size_t mad_linear_fp8_wgrad_workspace(long rows, int N, int K) {
    if (!wgrad_shape_ok(rows, N, K)) return 0;
    const size_t a = wgrad_workspace(wgrad_plan(rows, N, K, true), N, K), b = wgrad_workspace(wgrad_plan(rows, N, K, false), N, K);
    return a > b ? a : b;                       // whichever form the operands' alignment allows
}

template <int FMT, int T, int WN, int WK> static int launch_wgrad_tile(const F8WgradArgs& a, unsigned wgs, hipStream_t s) {
    constexpr int lds = F8Wg<T, T>::LDS;
    static int lds_dev = -1;
    auto kernel = &wgrad_fp8_tile_kernel<FMT, T, T, WN, WK>;
    MAD_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(kernel), lds, &lds_dev),
                "mad_linear_fp8_wgrad: cannot raise the dynamic LDS limit to %d", lds);
    hipLaunchKernelGGL((wgrad_fp8_tile_kernel<FMT, T, T, WN, WK>), dim3(wgs), dim3(64 * WN * WK), lds, s, a);
    return check_launch("mad_linear_fp8_wgrad");
}

extern "C" int mad_linear_fp8_wgrad(const void* dy, int dtype, const void* x, int x_type, const void* x_scale, float* dw, float* db,
                                    void* workspace, size_t workspace_bytes, long rows, int N, int K, int accumulate,
                                    int bias_accumulate, void* stream) {
    MAD_REQUIRE(dtype == MAD_BF16 || dtype == MAD_F32, "mad_linear_fp8_wgrad: bad dtype %d", dtype);
    MAD_REQUIRE(x_type == MAD_E4M3 || x_type == MAD_E5M2, "mad_linear_fp8_wgrad: x is of type %d, not an 8-bit one", x_type);
    MAD_REQUIRE(wgrad_shape_ok(rows, N, K), "mad_linear_fp8_wgrad: bad shape rows=%ld N=%d K=%d", rows, N, K);
    MAD_REQUIRE(dw && (rows == 0 || (dy && x && x_scale)), "mad_linear_fp8_wgrad: null pointer");
    MAD_REQUIRE(f8_aligned(x, x_scale), "mad_linear_fp8_wgrad: x must be 16-byte, its scales 4-byte aligned");
    const size_t need = mad_linear_fp8_wgrad_workspace(rows, N, K);
    MAD_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "mad_linear_fp8_wgrad: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    const bool tiled = wgrad_tiled(dy, dtype, N);
    const F8WgradPlan p = wgrad_plan(rows, N, K, tiled);
    const long wgs = (long)p.ntiles * p.ktiles * p.splits;
    MAD_REQUIRE(wgs <= 0x7fffffffL, "mad_linear_fp8_wgrad: N=%d K=%d need more workgroups than a launch holds", N, K);
    const size_t nk = (size_t)N * K;
    const bool join_w = p.splits > 1, join_b = db && (size_t)p.splits * p.ktiles > 1;
    float* part_w = (float*)workspace;
    float* part_b = part_w + (join_w ? (size_t)p.splits * nk : 0);
    F8WgradArgs a;
    a.dy = dy; a.x = (const unsigned char*)x; a.xs = (const unsigned char*)x_scale;
    a.dw = join_w ? part_w : dw;
    a.db = join_b ? part_b : db;
    a.M = rows; a.per = p.per; a.N = N; a.K = K;
    a.ntiles = p.ntiles; a.ktiles = p.ktiles; a.splits = p.splits;
    a.acc_w = accumulate; a.acc_b = !join_b && bias_accumulate;
    hipStream_t s = (hipStream_t)stream;
    int rc;
    if (tiled && p.tile == 256)
        rc = x_type == MAD_E4M3 ? launch_wgrad_tile<F8_E4M3, 256, 2, 4>(a, (unsigned)wgs, s) : launch_wgrad_tile<F8_E5M2, 256, 2, 4>(a, (unsigned)wgs, s);
    else if (tiled)
        rc = x_type == MAD_E4M3 ? launch_wgrad_tile<F8_E4M3, 128, 2, 2>(a, (unsigned)wgs, s) : launch_wgrad_tile<F8_E5M2, 128, 2, 2>(a, (unsigned)wgs, s);
    else {
#define LAUNCH(T, F) hipLaunchKernelGGL((wgrad_fp8_kernel<T, F>), dim3((unsigned)wgs), dim3(256), 0, s, a)
        if (dtype == MAD_BF16) { if (x_type == MAD_E4M3) LAUNCH(bf16_t, F8_E4M3); else LAUNCH(bf16_t, F8_E5M2); }
        else { if (x_type == MAD_E4M3) LAUNCH(float, F8_E4M3); else LAUNCH(float, F8_E5M2); }
#undef LAUNCH
        rc = check_launch("mad_linear_fp8_wgrad");
    }
    if (rc) return rc;
    if (join_w) {
        const size_t blocks = (nk + 255) / 256;
        hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s,
                           (const float*)part_w, dw, nk, p.splits, accumulate);
    }
    if (join_b)
        hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, (const float*)part_b, db,
                           (size_t)N, p.splits * p.ktiles, bias_accumulate);
    return join_w || join_b ? check_launch("mad_linear_fp8_wgrad") : 0;
}
