// Weight gradient of a layer whose input was kept in 8 bits (fp8.h):
//
//   dw[n][k] (+)= sum_m dy[m][n] * x[m][k]      db[n] (+)= sum_m dy[m][n]
//
// The scale of x changes along the reduction (one per row m), so the product cannot run on 8-bit operands; but bf16 holds
// every restored value exactly (to 2^-133, its smallest step), so x is widened on its way into LDS and the product runs on v_mfma_f32_16x16x32_bf16 without a
// further rounding.  dy is bf16, or fp32 cut into three bf16 terms whose sum is dy to 24 bits (x is exact, so three
// products give fp32 accuracy).  Both operands are stored with the reduction index slow and read with the transposing LDS
// read (ds_read_b64_tr_b16: a row of 16 lanes fetches 4 rows m x 16 columns, lane i receives column i).
// Shares of the rows write partial sums that a second kernel adds in share order: the result does not depend on timing.
//
// db is the gradient of an input column of ones: one more product per fragment of dy.  A workgroup makes it for every
// ktiles-th step only (kt = step mod ktiles), so that no tile of dw has more work than another; the parts are joined.
#include "fp8.h"
#include <math.h>

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
// step, two LDS stages.  dy comes by LDS-DMA one step ahead.  The bytes of x come by LDS-DMA two steps ahead into
// slots that only the lane that copied them reads (registers filled by ordinary loads had the compiler wait for them early), and are
// widened into the next stage between the products of this one, so that one barrier per step remains.  Columns past the end read
// what lies there, which only reaches results that are not stored; rows past the share are zeros (reads outside their buffer).
template <int BN, int BK> struct F8Wg {
    static constexpr int ROWS = 64, DY = ROWS * BN * 2, STAGE = DY + ROWS * BK * 2;
    static constexpr int RAW = ROWS * BK, SCALES = 2 * ROWS * 8;          // x as it comes; scales of two steps, two dwords per row
    static constexpr int LDS = 2 * STAGE + RAW + SCALES;
};

// The 16-byte chunk c of row m lies at c ^ swizzle(m): the eight rows that two lane groups read at a time, 32 bytes each, are in
// eight different parts of the 256 bytes that the banks span (with (m & 3) << 2 alone every read took twice as long).
__device__ __forceinline__ int swizzle(int m) { return ((m & 3) << 2) | ((m >> 2 & 1) << 1); }

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
        doff[j] = (unsigned)((4 * (c & 15) + lr) * a.N * 2 + (n0 + (c >> 4) * 128) * 2 + (((lane & 15) ^ swizzle(4 * wave + lr)) << 4));   // NW is even
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
    int turn = a.db ? 0 : -1;                                 // step mod ktiles

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
                    accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, frag(st, wn * (BN / WN) + 16 * (wk * FB + j), h), accb[j], 0, 0, 0);
        }
        if (a.db) turn = turn + 1 == a.ktiles ? 0 : turn + 1;
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
    if (a.db && g == 0) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            const int n = n0 + wn * (BN / WN) + 16 * (wk * FB + j) + r;
            if (n >= a.N) continue;
            float* p = a.db + ((size_t)split * a.ktiles + kt) * a.N + n;
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
// adds a partial sum to write and join.  The shares that balance the two, or fill the units once, and of the tiles the ones
// that come out shortest (us, 128 x 128 / 128 x 384 / 256 x 256: 65536 x 384 -> 1152 99 / 86 / 105, 16384 x 768 -> 2304
// 91 / 77 / 77, 8192 x 4096 -> 4096 319 / 388 / 234, 32768 x 256 -> 768 33 / 38 / 40).
struct F8WgradPlan { int bn, bk, ntiles, ktiles, splits; long per; double us; };

static F8WgradPlan wgrad_plan(long rows, int N, int K, bool tiled) {
    const long cus = f8_cus();
    auto plan = [&](int bn, int bk, int resident, double step_us) {
        F8WgradPlan p;
        p.bn = bn; p.bk = bk;
        p.ntiles = (N + bn - 1) / bn; p.ktiles = (K + bk - 1) / bk;
        const long tiles = (long)p.ntiles * p.ktiles, steps = (rows + 63) / 64;
        const double share_us = (double)N * K * 2.0e-6;                     // 8 bytes an element at 4 TB/s: written, then joined
        long s = (long)sqrt((double)steps * step_us / share_us + 1.0);
        const long most = resident * cus / tiles;
        if (s > most) s = most;
        if (s > steps) s = steps;
        p.splits = (int)(s < 1 ? 1 : s);
        p.per = ((rows + p.splits - 1) / p.splits + 63) / 64 * 64;
        const double rounds = (double)((tiles * p.splits + resident * cus - 1) / (resident * cus));
        p.us = rounds * (double)(p.per / 64) * step_us + (p.splits > 1 ? 3.0 + p.splits * share_us : 0.0);
        return p;
    };
    F8WgradPlan best = plan(128, 128, 2, 1.5);
    if (!tiled) return best;
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

template <int FMT, int BN, int BK, int WN, int WK> static int launch_wgrad_tile(const F8WgradArgs& a, unsigned wgs, hipStream_t s) {
    constexpr int lds = F8Wg<BN, BK>::LDS;
    static int lds_dev = -1;
    auto kernel = &wgrad_fp8_tile_kernel<FMT, BN, BK, WN, WK>;
    MAD_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(kernel), lds, &lds_dev),
                "mad_linear_fp8_wgrad: cannot raise the dynamic LDS limit to %d", lds);
    hipLaunchKernelGGL((wgrad_fp8_tile_kernel<FMT, BN, BK, WN, WK>), dim3(wgs), dim3(64 * WN * WK), lds, s, a);
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
#define TILE(BN, BK, WN, WK)                                                                                             \
    (x_type == MAD_E4M3 ? launch_wgrad_tile<F8_E4M3, BN, BK, WN, WK>(a, (unsigned)wgs, s)                                \
                        : launch_wgrad_tile<F8_E5M2, BN, BK, WN, WK>(a, (unsigned)wgs, s))
    if (tiled && p.bn == 256) rc = TILE(256, 256, 2, 4);
    else if (tiled && p.bk == 384) rc = TILE(128, 384, 2, 4);
    else if (tiled) rc = TILE(128, 128, 2, 2);
#undef TILE
    else {
#define LAUNCH(T, F) hipLaunchKernelGGL((wgrad_fp8_kernel<T, F>), dim3((unsigned)wgs), dim3(256), 0, s, a)
        if (dtype == MAD_BF16) { if (x_type == MAD_E4M3) LAUNCH(bf16_t, F8_E4M3); else LAUNCH(bf16_t, F8_E5M2); }
        else { if (x_type == MAD_E4M3) LAUNCH(float, F8_E4M3); else LAUNCH(float, F8_E5M2); }
#undef LAUNCH
        rc = check_launch("mad_linear_fp8_wgrad");
    }
    if (rc) return rc;
    if (!join_w && !join_b) return 0;
    F8JoinArgs j;
    j.part = part_w; j.dst = dw; j.part_b = part_b; j.dst_b = db;
    j.n = join_w ? nk : 0; j.nb = join_b ? N : 0; j.parts = p.splits; j.parts_b = p.splits * p.ktiles;
    j.acc = accumulate; j.acc_b = bias_accumulate;
    const size_t blocks = (j.n + 1023) / 1024;
    j.blocks = (int)(blocks < 4096 ? blocks : 4096);
    hipLaunchKernelGGL(wgrad_fp8_join_kernel, dim3((unsigned)(j.blocks + (j.nb + 255) / 256)), dim3(256), 0, s, j);
    return check_launch("mad_linear_fp8_wgrad");
}
