// Weight gradient of a layer whose input was kept in 8 bits (fp8.h):
//
//   dw[n][k] (+)= sum_m dy[m][n] * x[m][k]      db[n] (+)= sum_m dy[m][n]
//
// The scale of x changes along the reduction (one per row m), so the product cannot run on 8-bit operands; but bf16 holds
// every restored value exactly (to 2^-133, its smallest step), so x is widened on its way into LDS and the product runs on
// v_mfma_f32_16x16x32_bf16 without a further rounding.  dy is bf16, or fp32 cut into three bf16 terms whose sum is dy down
// to 2^-133 too, i.e. all 24 bits from 2^-109 on (x is exact, so three products give fp32 accuracy).  Both operands are stored with the reduction index slow and read with the
// transposing LDS read (ds_read_b64_tr_b16: a row of 16 lanes fetches 4 rows m x 16 columns, lane i receives column i).
// Shares of the rows write partial sums that a second kernel adds in share order: the result does not depend on timing.
//
// db is the gradient of an input column of ones: one more product per fragment of dy.  A workgroup makes it for every
// ktiles-th step only (kt = step mod turns, turns = ktiles), so that no tile of dw has more work than another; the parts are
// joined.  Where that would be all there is to join, and the launch costs more than the sixteenth it saves, turns is 1.
#include "fp8.h"
#include <math.h>

namespace mad {

struct F8WgradArgs {
    const void* dy; const unsigned char* x; const unsigned char* xs;
    float* dw; float* db;                      // destinations, or partial slabs when splits > 1
    long M, per;                               // rows, rows per share (a multiple of 32)
    int N, K, ntiles, ktiles, splits, turns, acc_w, acc_b;
};

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

__device__ __forceinline__ bf16x8 tr_pair(const unsigned char* lo, const unsigned char* hi) {
    const bf16x4 l = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)lo);
    const bf16x4 h = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)hi);
    return bf16x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
}

// The 16-byte chunk c of row m lies at c ^ swizzle(m): the eight rows that two lane groups read at a time, 32 bytes each, are in
// eight different parts of the 256 bytes that the banks span (with (m & 3) << 2 alone every read took twice as long).
__device__ __forceinline__ int swizzle(int m) { return ((m & 3) << 2) | ((m >> 2 & 1) << 1); }

// Eight elements of dy on their way to bf16.  fp32 is cut into three terms by truncation, 8 bits of the 24 each, so that every
// difference is exact; of a value that is not finite the first term is all (truncated, a NaN keeps a set bit).
template <typename T> struct DyPiece;
template <> struct DyPiece<bf16_t> {
    uint4 v;
    __device__ __forceinline__ void clear() { v = uint4{0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const bf16_t* p) { Piece8<bf16_t> t; t.load(p); v = __builtin_bit_cast(uint4, t.v); }
    __device__ __forceinline__ void load_some(const bf16_t* p, int n) {
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = (2 * e < n ? (unsigned)p[2 * e] : 0u) | (2 * e + 1 < n ? (unsigned)p[2 * e + 1] << 16 : 0u);
        v = uint4{w[0], w[1], w[2], w[3]};
    }
    __device__ __forceinline__ void terms(uint4* o) const { o[0] = v; }
};
template <> struct DyPiece<float> {
    float f[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.0f;
    }
    __device__ __forceinline__ void load(const float* p) { load8<float>(p, f); }
    __device__ __forceinline__ void load_some(const float* p, int n) { load8_tail<float>(p, 0, n, f); }
    __device__ __forceinline__ void terms(uint4* o) const {
        unsigned t[3][8], top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) { const unsigned u = __float_as_uint(f[e]) & 0x7fffffffu; top = u > top ? u : top; }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[0][e] = __float_as_uint(f[e]);
            const float r = f[e] - __uint_as_float(t[0][e] & 0xffff0000u);
            t[1][e] = __float_as_uint(r);
            t[2][e] = __float_as_uint(r - __uint_as_float(t[1][e] & 0xffff0000u));
        }
        if (__any(top >= 0x7f800000u)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned u = t[0][e] & 0x7fffffffu;
                if (u >= 0x7f800000u) { t[0][e] |= u > 0x7f800000u ? 0x400000u : 0u; t[1][e] = t[2][e] = 0; }
            }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            unsigned* w = &o[p].x;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(t[p][2 * e + 1], t[p][2 * e], 0x07060302u);
        }
    }
};

// General form: dy in fp32, or in bf16 with rows that start anywhere.  128 (n) x BK (k) of dw per workgroup, 32 rows m per step,
// waves of 64 x 64; LDS [32 rows][128 columns] bf16 per term of dy and per 128 columns of x, two stages.  Both operands pass
// through registers: loaded a step and a half ahead, cut or widened between the two halves of the products of the step before.
// As in the tiled form below, columns past the end hold whatever follows in memory, rows past the share zeros.
// 8192 x 4096 -> 4096: fp32 808 us (three products: 1020 TFLOP/s of the matrix units; with one stage, loads inside the step and
// terms rounded to nearest 1677), bf16 into 4095 columns 438 (1394).
template <typename T, int BK> struct F8WgGeneral {
    static constexpr int NP = sizeof(T) == 4 ? 3 : 1, TILE = 32 * 256, STAGE = (NP + BK / 128) * TILE, LDS = 2 * STAGE;
};

template <typename T, int FMT, int BK>
__global__ __launch_bounds__(2 * BK) void wgrad_fp8_kernel(F8WgradArgs a) {
    using L = F8WgGeneral<T, BK>;
    constexpr int NP = L::NP, TILE = L::TILE, WK = BK / 64, FB = 4 / WK, DP = 256 / BK;
    static_assert(BK == 128 || BK == 256, "tile");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / WK, wk = wave % WK;
    const int tiles = a.ntiles * a.ktiles;
    const int split = blockIdx.x / tiles, t = blockIdx.x - split * tiles;
    const int nt = t / a.ktiles, kt = t - nt * a.ktiles;
    const int n0 = nt * 128, k0 = kt * BK;
    const long m_begin = (long)split * a.per, m_end = m_begin + a.per < a.M ? m_begin + a.per : a.M;
    const int steps = (int)((m_end - m_begin + 31) / 32);
    const int xp = f8_pitch(a.K), sp = f8_scale_pitch(a.K);
    const size_t total = (size_t)a.M * a.N;

    // this thread's pieces of a step: DP times eight columns of dy, sixteen of x
    const int dr = tid >> 4, dc = 8 * (tid & 15), xr = tid / (BK / 16), xc = 16 * (tid % (BK / 16));
    DyPiece<T> dv[DP];
    uint4 xv;
    float sc;
    auto fetch = [&](int s) {
        const long m = m_begin + 32L * s;
#pragma unroll
        for (int h = 0; h < DP; ++h) {
            const long mr = m + dr + 16 * h;
            const size_t at = (size_t)mr * a.N + n0 + dc;
            dv[h].clear();
            if (mr < m_end && n0 + dc < a.N) {
                if (at + 8 <= total) dv[h].load((const T*)a.dy + at);
                else dv[h].load_some((const T*)a.dy + at, a.N - n0 - dc);
            }
        }
        xv = uint4{0, 0, 0, 0};
        sc = 1.0f;
        if (m + xr < m_end && k0 + xc < xp) {
            xv = *reinterpret_cast<const uint4*>(a.x + (size_t)(m + xr) * xp + k0 + xc);
            sc = f8_scale(a.xs[(size_t)(m + xr) * sp + (k0 + xc) / F8_BLOCK]);
        }
    };
    auto put = [&](int buf) {
        unsigned char* st = smem + buf * L::STAGE;
#pragma unroll
        for (int h = 0; h < DP; ++h) {
            const int row = dr + 16 * h;
            unsigned char* d = st + row * 256 + (((dc >> 3) ^ swizzle(row)) << 4);
            uint4 o[NP];
            dv[h].terms(o);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4*>(d + p * TILE) = o[p];
        }
        unsigned char* d = st + (NP + xc / 128) * TILE + xr * 256;
        const int chunk = (xc % 128 >> 3) ^ swizzle(xr);
        *reinterpret_cast<bf16x8*>(d + (chunk << 4)) = f8_bf16x8<FMT>(xv.x, xv.y, sc);
        *reinterpret_cast<bf16x8*>(d + ((chunk ^ 1) << 4)) = f8_bf16x8<FMT>(xv.z, xv.w, sc);
    };

    f32x4 acc[4][4], accb[FB];                                // [k fragment][n fragment]
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < FB; ++j) accb[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const __bf16 one = (__bf16)1.0f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};
    int turn = a.db ? 0 : -1;                                 // step mod turns

    const int g = lane >> 4, q = (lane >> 2) & 3, pp = lane & 3;
    const int frow = (4 * g + q) * 256 + (pp & 1) * 8, fswz = swizzle(4 * g + q);
    auto frag = [&](const unsigned char* tile, int col) {     // 16 columns from col, all 32 rows
        const unsigned char* p = tile + frow + ((((col >> 3) + (pp >> 1)) ^ fswz) << 4);
        return tr_pair(p, p + 16 * 256);
    };

    fetch(0);
    put(0);
    fetch(1);
    for (int s = 0; s < steps; ++s) {
        __syncthreads();                   // step s is visible; every wave is done with the stage refilled below
        const unsigned char* st = smem + (s & 1) * L::STAGE;
        if (turn == kt) {
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int j = 0; j < FB; ++j)
                    accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, frag(st + p * TILE, wn * 64 + 16 * (wk * FB + j)), accb[j],
                                                                      0, 0, 0);
        }
        if (a.db) turn = turn + 1 == a.turns ? 0 : turn + 1;
        bf16x8 xf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xf[i] = frag(st + (NP + wk / 2) * TILE, wk % 2 * 64 + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j == 2) { put((s + 1) & 1); fetch(s + 2); }
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const bf16x8 d = frag(st + p * TILE, wn * 64 + 16 * j);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], d, acc[i][j], 0, 0, 0);
            }
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
            if (k >= a.K) continue;
            float* p = dw + (size_t)n * a.K + k;
            f32x4 v = acc[i][j];
            if (direct && a.acc_w) v += load4_tail<float>(p, k, a.K);
            store4_tail<float>(p, k, a.K, v);
        }
    }
    if (a.db && g == 0 && kt < a.turns) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int n = n0 + wn * 64 + 16 * (wk * FB + j) + r;
            if (n >= a.N) continue;
            float* p = a.db + ((size_t)split * a.turns + kt) * a.N + n;
            *p = (a.acc_b ? *p : 0.0f) + accb[j][0];
        }
    }
}

// Tiled form: dy in bf16 with rows of whole 16-byte pieces.  BN (n) x BK (k) of dw per workgroup of WN x WK waves, 64 rows m per
// step, two LDS stages.  dy comes by LDS-DMA one step ahead.  The bytes of x come by LDS-DMA two steps ahead into
// slots that only the lane that copied them reads (registers filled by ordinary loads had the compiler wait for them early), and are
// widened into the next stage between the products of this one, so that one barrier per step remains.  Columns past the end read
// what lies there, which only reaches results that are not stored; rows past the share are zeros (reads outside their buffer).
// 8192 x 4096 -> 4096 247 us, 1110 TFLOP/s (a library's bf16 product of 8192^3: 1383).  A step of 64 rows and 256 x 256 is 2048 cycles of
// products and 295 KB through LDS (197 of them fragments, the rest copies in and x read and written to widen it), 2300 cycles at 128
// bytes each.  It takes 4600 cycles, about their sum: neither pipe is the bound by itself, the two hardly overlap.
template <int BN, int BK> struct F8Wg {
    static constexpr int ROWS = 64, DY = ROWS * BN * 2, STAGE = DY + ROWS * BK * 2;
    static constexpr int RAW = ROWS * BK, SCALES = 2 * ROWS * 8;          // x as it comes; scales of two steps, two dwords per row
    static constexpr int LDS = 2 * STAGE + RAW + SCALES;
};

template <int FMT, int BN, int BK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) void wgrad_fp8_tile_kernel(F8WgradArgs a) {
    using L = F8Wg<BN, BK>;
    constexpr int NW = WN * WK, FN = BN / WN / 16, FK = BK / WK / 16;
    constexpr int FB = FN / WK;                                           // column sums: the waves of a row share its fragments
    constexpr int DPW = BN / 8 / NW;                                      // dy copies per wave and step (4 rows x 128 columns each)
    constexpr int XPT = 64 * BK / 16 / (64 * NW);                         // 16-byte pieces of x per thread and step
    static_assert(BK <= 512 && (BK <= 256 || BK == 384) && NW % 2 == 0 && BN % 128 == 0 && BK % 128 == 0 && BN % (8 * NW) == 0 &&
                  XPT * 16 * NW == BK && FN % WK == 0, "tile");
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
    const int xp = f8_pitch(a.K), sp = f8_scale_pitch(a.K);

    // where this lane's copies read: offsets inside the 64 rows of a step
    const int lr = lane >> 4;
    unsigned doff[DPW];
#pragma unroll
    for (int j = 0; j < DPW; ++j) {
        const int c = j * NW + wave;                                      // half c / 16, rows 4 (c % 16) ..
        doff[j] = (unsigned)((4 * (c & 15) + lr) * a.N * 2 + (n0 + (c >> 4) * 128) * 2 +
                             (((lane & 15) ^ swizzle(4 * wave + lr)) << 4));                  // (NW is even)
    }
    unsigned xoff[XPT];
    int xdst[XPT], sbyte[XPT], odd = 0;
#pragma unroll
    for (int u = 0; u < XPT; ++u) {
        const int i = u * 64 * NW + tid, row = i / (BK / 16), piece = i % (BK / 16), half = piece >> 3;
        xoff[u] = (unsigned)(row * xp + k0 + 16 * piece);
        // the row's dword of scales that holds the block: the first of the tile's, or the one behind it
        const int block = (k0 / F8_BLOCK & 3) + half;
        sbyte[u] = (block >> 2) * L::ROWS * 4 + row * 4 + (block & 3);
        odd |= (row & 1) << u;
        // odd rows write their second piece first: the pieces of a write then cover all banks
        xdst[u] = L::DY + (half * L::ROWS + row) * 256 + (((2 * (piece & 7) + (row & 1)) ^ swizzle(row)) << 4);
    }
    const unsigned lds0 = lds_addr(smem);
    // rows of step s that exist (none behind the last: the reads then deliver zeros)
    auto step_rows = [&](int s) {
        const long left = m_end - m_begin - (long)s * L::ROWS;
        return left < 0 ? 0 : left < L::ROWS ? (int)left : L::ROWS;
    };
    auto fetch_dy = [&](int s, int buf) {                                 // dy of step s into its stage
        const long m = m_begin + (long)s * L::ROWS;
        const u32x4 db = f8_buffer((const unsigned char*)a.dy + (size_t)m * a.N * 2, (unsigned)(step_rows(s) * a.N * 2));
#pragma unroll
        for (int j = 0; j < DPW; ++j) buf_lds16(db, doff[j], 0, lds0 + buf * L::STAGE + (j * NW + wave) * 1024);
    };
    constexpr int RAW = 2 * L::STAGE, SCALES = RAW + L::RAW;
    // scales of step s: the dword of each row that holds the tile's first block and, where the tile may reach past it, the next
    auto fetch_scales = [&](int s) {
        const long m = m_begin + (long)s * L::ROWS;
        const u32x4 sb = f8_buffer(a.xs + (size_t)m * sp, (unsigned)(step_rows(s) * sp));
        const int first = k0 / F8_BLOCK & ~3;
        const unsigned dst = lds0 + SCALES + (s & 1) * L::ROWS * 8;
        if (wave == NW - 1) buf_lds4(sb, (unsigned)(lane * sp + first), 0, dst);
        if (BK > 256 && wave == NW - 2) buf_lds4(sb, first + 4 < sp ? (unsigned)(lane * sp + first + 4) : F8_OUTSIDE, 0, dst + L::ROWS * 4);
    };
    auto fetch_x = [&](int s) {                                           // x of step s into this lane's slots
        const long m = m_begin + (long)s * L::ROWS;
        const u32x4 xb = f8_buffer(a.x + (size_t)m * xp, (unsigned)(step_rows(s) * xp));
#pragma unroll
        for (int u = 0; u < XPT; ++u) {
            buf_lds16(xb, xoff[u], 0, lds0 + RAW + (u * NW + wave) * 1024);
        }
    };
    auto widen = [&](int s, int buf) {                                    // the fetched x of step s into the stage
        unsigned char* d = smem + buf * L::STAGE;
#pragma unroll
        for (int u = 0; u < XPT; ++u) {
            const uint4 v = *reinterpret_cast<const uint4*>(smem + RAW + (u * 64 * NW + tid) * 16);
            const float sc = f8_scale(smem[SCALES + (s & 1) * L::ROWS * 8 + sbyte[u]]);
            const bool o = odd >> u & 1;
            const unsigned a0 = o ? v.z : v.x, a1 = o ? v.w : v.y, b0 = o ? v.x : v.z, b1 = o ? v.y : v.w;
            *reinterpret_cast<bf16x8*>(d + xdst[u]) = f8_bf16x8<FMT>(a0, a1, sc);
            *reinterpret_cast<bf16x8*>(d + (xdst[u] ^ 16)) = f8_bf16x8<FMT>(b0, b1, sc);
        }
    };

    f32x4 acc[FK][FN], accb[FB];                              // [k fragment][n fragment]
#pragma unroll
    for (int j = 0; j < FB; ++j) accb[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < FN; ++j) {
#pragma unroll
        for (int i = 0; i < FK; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const __bf16 one = (__bf16)1.0f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};
    int turn = a.db ? 0 : -1;                                 // step mod turns

    // fragment of 16 columns: rows 4g + q and 16 rows on, 8 bytes at columns 4 pp
    const int frow = (4 * g + q) * 256 + (pp & 1) * 8, fswz = swizzle(4 * g + q);
    auto frag = [&](const unsigned char* tile, int c, int h) {
        const int chunk = ((c & 127) >> 3) + (pp >> 1);
        const unsigned char* p = tile + (c >> 7) * L::ROWS * 256 + h * 32 * 256 + frow + ((chunk ^ fswz) << 4);
        return tr_pair(p, p + 16 * 256);
    };

    fetch_scales(0);
    fetch_x(0);
    fetch_scales(1);
    dma_wait_all();
    __syncthreads();
    fetch_dy(0, 0);
    widen(0, 0);
    fetch_x(1);
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        dma_wait_all();
        __syncthreads();                   // step s is visible; every wave is done with the stage refilled below
        fetch_dy(s + 1, buf ^ 1);
        fetch_scales(s + 2);
        const unsigned char* st = smem + buf * L::STAGE;
        if (turn == kt) {                  // not among the products below: a branch around each would keep their reads from running ahead
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < FB; ++j)
                    accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, frag(st, wn * (BN / WN) + 16 * (wk * FB + j), h), accb[j],
                                                                      0, 0, 0);
        }
        if (a.db) turn = turn + 1 == a.turns ? 0 : turn + 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 xf[FK], d[FN];
#pragma unroll
            for (int i = 0; i < FK; ++i) xf[i] = frag(st + L::DY, wk * (BK / WK) + 16 * i, h);
#pragma unroll
            for (int j = 0; j < FN; ++j) d[j] = frag(st, wn * (BN / WN) + 16 * j, h);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FK; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i], d[j], acc[i][j], 0, 0, 0);
            if (h == 0) {                  // between the products of the other waves
                widen(s + 1, buf ^ 1);
                fetch_x(s + 2);
            }
        }
    }
    dma_wait_all();                        // the copies of the step behind the last

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
    }
    if (a.db && g == 0 && kt < a.turns) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int n = n0 + wn * (BN / WN) + 16 * (wk * FB + j) + r;
            if (n >= a.N) continue;
            float* p = a.db + ((size_t)split * a.turns + kt) * a.N + n;
            *p = (a.acc_b ? *p : 0.0f) + accb[j][0];
        }
    }
}

// dw[i] (+)= sum of `parts` partial sums of n elements, in order; the last workgroups do the same for db (nb elements of
// `parts_b`).  Four elements per thread and eight parts in flight: the loads, not the additions, take the time.
struct F8JoinArgs { const float* part; float* dst; const float* part_b; float* dst_b; size_t n; int nb, parts, parts_b, acc, acc_b, blocks; };

__global__ __launch_bounds__(256) void wgrad_fp8_join_kernel(F8JoinArgs a) {
    if ((int)blockIdx.x >= a.blocks) {
        const int i = (blockIdx.x - a.blocks) * 256 + threadIdx.x;
        if (i >= a.nb) return;
        float s = 0.0f;
#pragma unroll 8
        for (int z = 0; z < a.parts_b; ++z) s += a.part_b[(size_t)z * a.nb + i];
        a.dst_b[i] = a.acc_b ? a.dst_b[i] + s : s;
        return;
    }
    for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4; i < a.n; i += (size_t)a.blocks * 1024) {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (i + 4 <= a.n) {
            typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 8
            for (int z = 0; z < a.parts; ++z) s += *reinterpret_cast<const f32x4u*>(a.part + (size_t)z * a.n + i);
            if (a.acc) s += load4_tail<float>(a.dst + i, 0, 4);
            store4_tail<float>(a.dst + i, 0, 4, s);
        } else {
            for (size_t e = i; e < a.n; ++e) {
                float v = 0.0f;
                for (int z = 0; z < a.parts; ++z) v += a.part[(size_t)z * a.n + e];
                a.dst[e] = a.acc ? a.dst[e] + v : v;
            }
        }
    }
}

// How a gradient is cut: the form, its tiles and the shares of the rows.  A step of 64 rows takes a workgroup about 1.5 us with tiles of
// 128 x 128 (two workgroups to a unit), 1.9 with 128 x 384 and 1.85 with 256 x 256; a share more shortens the rows of each and
// adds a partial sum to write and join.  The general form takes 1.7 us (bf16; 128 x 256 is no faster there) and 3.5 (fp32; 3.15 with
// 128 x 256, one workgroup: 16384 x 2048 -> 2048 483 / 428 us, 65536 x 128 -> 384 48 / 53).  The shares that balance the two, or fill
// the units once, and of the tiles the ones that come out shortest (us, 128 x 128 / 128 x 384 / 256 x 256: 65536 x 384 -> 1152
// 99 / 86 / 105, 16384 x 768 -> 2304 91 / 77 / 77, 8192 x 4096 -> 4096 319 / 388 / 245, 32768 x 256 -> 768 33 / 38 / 40).
enum F8WgradForm { WG_TILED, WG_BF16, WG_F32 };
struct F8WgradPlan { int bn, bk, ntiles, ktiles, splits, turns; long per; double us; };

static F8WgradPlan wgrad_plan(long rows, int N, int K, F8WgradForm form) {
    const long cus = f8_cus();
    auto plan = [&](int bn, int bk, int resident, double step_us) {
        const double share_us = (double)N * K * 2.0e-6;                     // 8 bytes an element at 4 TB/s: written, then joined
        const double join_us = 5.0;                                         // another launch, for GPU and host
        const long steps = (rows + 63) / 64;
        auto with = [&](long s) {
            F8WgradPlan p;
            p.bn = bn; p.bk = bk;
            p.ntiles = (N + bn - 1) / bn; p.ktiles = (K + bk - 1) / bk;
            p.splits = (int)s;
            p.per = ((rows + s - 1) / s + 63) / 64 * 64;
            const double rounds = (double)(((long)p.ntiles * p.ktiles * s + resident * cus - 1) / (resident * cus));
            p.us = rounds * (double)(p.per / 64) * step_us;
            p.turns = s == 1 && p.us < 16 * join_us ? 1 : p.ktiles;
            if (s > 1) p.us += join_us + s * share_us;
            return p;
        };
        const F8WgradPlan one = with(1);
        long s = (long)sqrt((double)steps * step_us / share_us + 1.0);
        const long most = resident * cus / ((long)one.ntiles * one.ktiles);
        if (s > most) s = most;
        if (s > steps) s = steps;
        if (s < 2) return one;
        const F8WgradPlan many = with(s);
        return many.us < one.us ? many : one;
    };
    if (form == WG_BF16) return plan(128, 128, 2, 1.7);
    if (form == WG_F32) {
        const F8WgradPlan small = plan(128, 128, 2, 3.5), wide = plan(128, 256, 1, 3.15);
        return wide.us < small.us ? wide : small;
    }
    F8WgradPlan best = plan(128, 128, 2, 1.5);
    for (const F8WgradPlan& p : {plan(128, 384, 1, 1.9), plan(256, 256, 1, 1.85)})
        if (p.us < best.us) best = p;
    return best;
}

}  // namespace mad

using namespace mad;

static bool wgrad_shape_ok(long rows, int N, int K) {
    return rows >= 0 && N > 0 && N <= MAD_FP8_MAX_WIDTH && K > 0 && K <= MAD_FP8_MAX_WIDTH;
}

static size_t wgrad_workspace(const F8WgradPlan& p, int N, int K) {
    const size_t w = p.splits > 1 ? (size_t)p.splits * N * K : 0;
    const size_t b = (size_t)p.splits * p.turns > 1 ? (size_t)p.splits * p.turns * N : 0;
    return (w + b) * sizeof(float);
}

// LDS-DMA of dy needs rows of whole 16-byte pieces
static F8WgradForm wgrad_form(const void* dy, int dtype, int N) {
    return dtype == MAD_F32 ? WG_F32 : N % 8 == 0 && !((uintptr_t)dy & 15) ? WG_TILED : WG_BF16;
}

extern "C" size_t mad_linear_fp8_wgrad_workspace(long rows, int N, int K) {
    if (!wgrad_shape_ok(rows, N, K)) return 0;
    size_t most = 0;                            // of the forms: which one runs depends on the operands' type and alignment
    for (const F8WgradForm f : {WG_TILED, WG_BF16, WG_F32}) {
        const size_t n = wgrad_workspace(wgrad_plan(rows, N, K, f), N, K);
        if (n > most) most = n;
    }
    return most;
}

static int launch_wgrad(void (*kernel)(F8WgradArgs), int lds, int* lds_dev, int threads, const F8WgradArgs& a, unsigned wgs, hipStream_t s) {
    MAD_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(kernel), lds, lds_dev),
                "mad_linear_fp8_wgrad: cannot raise the dynamic LDS limit to %d", lds);
    hipLaunchKernelGGL(kernel, dim3(wgs), dim3(threads), lds, s, a);
    return check_launch("mad_linear_fp8_wgrad");
}

template <int FMT> static int launch_wgrad(F8WgradForm form, const F8WgradPlan& p, const F8WgradArgs& a, hipStream_t s) {
    const unsigned wgs = (unsigned)(p.ntiles * p.ktiles * p.splits);
#define TILE(BN, BK, WN, WK)                                                                                               \
    { static int dev = -1; return launch_wgrad(&wgrad_fp8_tile_kernel<FMT, BN, BK, WN, WK>, F8Wg<BN, BK>::LDS, &dev, 64 * WN * WK, a, wgs, s); }
#define GENERAL(T, BK)                                                                                                     \
    { static int dev = -1; return launch_wgrad(&wgrad_fp8_kernel<T, FMT, BK>, F8WgGeneral<T, BK>::LDS, &dev, 2 * BK, a, wgs, s); }
    if (form == WG_F32) { if (p.bk == 256) GENERAL(float, 256) else GENERAL(float, 128) }
    if (form == WG_BF16) GENERAL(bf16_t, 128)
    if (p.bn == 256) TILE(256, 256, 2, 4)
    if (p.bk == 384) TILE(128, 384, 2, 4)
    TILE(128, 128, 2, 2)
#undef TILE
#undef GENERAL
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
    const F8WgradForm form = wgrad_form(dy, dtype, N);
    const F8WgradPlan p = wgrad_plan(rows, N, K, form);
    const long wgs = (long)p.ntiles * p.ktiles * p.splits;
    MAD_REQUIRE(wgs <= 0x7fffffffL, "mad_linear_fp8_wgrad: N=%d K=%d need more workgroups than a launch holds", N, K);
    const size_t nk = (size_t)N * K;
    const bool join_w = p.splits > 1, join_b = db && (size_t)p.splits * p.turns > 1;
    float* part_w = (float*)workspace;
    float* part_b = part_w + (join_w ? (size_t)p.splits * nk : 0);
    F8WgradArgs a;
    a.dy = dy; a.x = (const unsigned char*)x; a.xs = (const unsigned char*)x_scale;
    a.dw = join_w ? part_w : dw;
    a.db = join_b ? part_b : db;
    a.M = rows; a.per = p.per; a.N = N; a.K = K;
    a.ntiles = p.ntiles; a.ktiles = p.ktiles; a.splits = p.splits; a.turns = p.turns;
    a.acc_w = accumulate; a.acc_b = !join_b && bias_accumulate;
    hipStream_t s = (hipStream_t)stream;
    const int rc = x_type == MAD_E4M3 ? launch_wgrad<F8_E4M3>(form, p, a, s) : launch_wgrad<F8_E5M2>(form, p, a, s);
    if (rc) return rc;
    if (!join_w && !join_b) return 0;
    F8JoinArgs j;
    j.part = part_w; j.dst = dw; j.part_b = part_b; j.dst_b = db;
    j.n = join_w ? nk : 0; j.nb = join_b ? N : 0; j.parts = p.splits; j.parts_b = p.splits * p.turns;
    j.acc = accumulate; j.acc_b = bias_accumulate;
    const size_t blocks = (j.n + 1023) / 1024;
    j.blocks = (int)(blocks < 4096 ? blocks : 4096);
    hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)(j.blocks + (j.nb + 255) / 256)), dim3(256), 0, s, j);
    return check_launch("mad_linear_fp8_wgrad");
}
