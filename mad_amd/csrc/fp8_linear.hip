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
#include <type_traits>

namespace mad {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct F8LinArgs {
    const void* x; const unsigned char* xs;        // x as bytes with scales, or as bf16 / fp32 (xs null)
    const unsigned char* w; const unsigned char* ws;
    const float* bias; const void* residual; void* y;
    unsigned char* q; unsigned char* scale;        // direct form: where the rounded x is kept, or null
    long M;
    int K, N, mtiles, ntiles;
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
    if (a.bias) v += load4_tail<float>(a.bias + n, n, a.N);
    if (a.residual) v += load4_tail<TO>((const TO*)a.residual + m * a.N + n, n, a.N);
    store4_tail<TO>((TO*)a.y + m * a.N + n, n, a.N, v);
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

// rows of x that start, and end, with whole 16-byte pieces
__host__ __device__ __forceinline__ bool whole_pieces(const void* x, int dtype, int K) {
    return K % (dtype == MAD_BF16 ? 8 : 4) == 0 && ((uintptr_t)x & 15) == 0;
}

// Lanes come in pairs with rows r and r + 1.  Each has loaded a piece of both, so that a load of the wave touches eight rows, a whole
// line of each: even lanes keep that of r and pass on the other, odd lanes the other way round.  (With 16 rows and half a line of
// each to a load, us: packed 256 x 2048 -> 2048 11.3 / 8.2 in pairs, fp32 16 x 4096 -> 8192 15.5 / 11.6.)
__device__ __forceinline__ void swap_pair(bool odd, unsigned& a, unsigned& b) {
    const unsigned t = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(odd ? a : b), 0xB1, 0xF, 0xF, true);     // lane ^ 1
    a = odd ? t : a;
    b = odd ? b : t;
}

// Direct form: operands from global memory straight into registers, (16 MF) x (16 NF) outputs per workgroup, its NW
// waves taking every NW-th block of the reduction.  Few rows are bound by the latency of reading the weights once, so the reduction
// is spread over many waves; their sums are joined through LDS pairwise, wave w and w + NW/2 first: a fixed order.  x may come
// unpacked: it is rounded to XF on its way in, by every workgroup that needs it, and kept in memory by the first of them if asked.
// Measured: 1 x 768 -> 768 2.6 us packed, 3.3 from bf16 (a launch); 32 x 4096 -> 8192 from bf16 12.1 with the weights in the
// last-level cache (2.8 TB/s), 16.6 with none there.  Loading a block ahead of the products gained nothing and cost the forms that
// round x their registers; so did starting the workgroups at different blocks.
template <int XK, int XF, typename TO, int MF, int NF, int NW>
__global__ __launch_bounds__(64 * NW) void linear_fp8_direct_kernel(F8LinArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 red[NW / 2][MF * NF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const long mt = blockIdx.x / a.ntiles;
    const int nt = (int)(blockIdx.x - mt * a.ntiles);
    const long m0 = mt * (16 * MF);
    const int n0 = nt * (16 * NF);
    const int kb = f8_blocks(a.K), wp = f8_pitch(a.K), sp = f8_scale_pitch(a.K);

    // Buffer loads without a branch: lanes behind the last row, or behind the end of their row, read zeros.
    const int mrem = a.M - m0 < 16 * MF ? (int)(a.M - m0) : 16 * MF, nrem = a.N - n0 < 16 * NF ? a.N - n0 : 16 * NF;
    const auto wbuf = f8_resource(a.w + (size_t)n0 * wp, nrem * wp);
    const auto wsbuf = f8_resource(a.ws + (size_t)(n0 / F8_BLOCK) * sp, f8_blocks(n0 % F8_BLOCK + nrem) * sp);
    constexpr int XB = XK < X_BF16 ? 1 : XK == X_BF16 ? 2 : 4;
    const int xpitch = XK < X_BF16 ? wp : a.K * XB;
    const auto xbuf = f8_resource((const unsigned char*)a.x + (size_t)m0 * xpitch, mrem * xpitch);
    const auto xsbuf = f8_resource(a.xs + (XK < X_BF16 ? (size_t)m0 * sp : 0), XK < X_BF16 ? mrem * sp : 0);
    const bool whole = XK >= X_BF16 && whole_pieces(a.x, XK == X_BF16 ? MAD_BF16 : MAD_F32, a.K);
    auto load16 = [](const auto& rsrc, int off) { return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0)); };

    f32x4 acc[NF][MF];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // a lane's 32 bytes of a block are chunks g and g + 4 of its row
    const bool odd = r & 1;
    auto fragment = [&](const auto& rsrc, int row0, int kt) {
        const int c = kt * F8_BLOCK + 64 * (r & 1) + 16 * g, off = (row0 + (r & ~1)) * wp + c;
        uint4 v = load16(rsrc, c < wp ? off : (int)F8_OUTSIDE), w = load16(rsrc, c < wp ? off + wp : (int)F8_OUTSIDE);
        swap_pair(odd, v.x, w.x); swap_pair(odd, v.y, w.y); swap_pair(odd, v.z, w.z); swap_pair(odd, v.w, w.w);
        return pair16(v, w);
    };
#pragma unroll 1
    for (int kt = wave; kt < kb; kt += NW) {
        const int c = kt * F8_BLOCK + 16 * g;
        i32x8 wf[NF];
        int wsc[NF];
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            wf[j] = fragment(wbuf, 16 * j, kt);
            wsc[j] = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(wsbuf, ((n0 % F8_BLOCK + 16 * j + r) / F8_BLOCK) * sp + kt, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            i32x8 xf;
            int xsc;
            if constexpr (XK < X_BF16) {
                xf = fragment(xbuf, 16 * i, kt);
                xsc = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(xsbuf, (16 * i + r) * sp + kt, 0, 0);
            } else {
                using T = typename std::conditional<XK == X_BF16, bf16_t, float>::type;
                // unpacked: pieces q of eight columns, 0 and 1 of the pair's even row, 2 and 3 of its odd one
                const int c8 = kt * F8_BLOCK + 16 * g + 8 * (r & 1), row0 = 16 * i + (r & ~1);
                auto reduce = [](unsigned v, auto top) {                   // over the eight lanes that hold a row
                    v = top(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
                    v = top(v, __shfl_xor(v, 16));
                    return top(v, __shfl_xor(v, 32));
                };
                int sc[2];
                if (XK == X_BF16 && whole) {
                    // on pairs of bf16 as they are: their magnitudes' maximum as 16-bit integers, and one conversion for two
                    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
                    auto top16 = [](unsigned a, unsigned b) {
                        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
                    };
                    uint4 v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int col = c8 + 64 * (q & 1);
                        v[q] = load16(xbuf, col < a.K ? (row0 + (q >> 1)) * xpitch + 2 * col : (int)F8_OUTSIDE);
                    }
                    const unsigned* w = &v[0].x;
                    unsigned m[2] = {0, 0};
#pragma unroll
                    for (int e = 0; e < 16; ++e) m[e >> 3] = top16(m[e >> 3], w[e] & 0x7fff7fffu);
                    // of the even row in the low half, of the odd one in the high half
                    unsigned u = top16(m[0] & 0xffffu, m[0] >> 16) | top16(m[1] & 0xffffu, m[1] >> 16) << 16;
                    if (__any((u & 0xffffu) >= 0x7f80u || u >= 0x7f800000u)) {     // something is not finite: it does not count
                        unsigned f[2] = {0, 0};
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const unsigned lo = w[e] & 0x7fffu, hi = w[e] >> 16 & 0x7fffu;
                            unsigned& t = f[e >> 3];
                            t = lo < 0x7f80u && lo > t ? lo : t;
                            t = hi < 0x7f80u && hi > t ? hi : t;
                        }
                        u = f[0] | f[1] << 16;
                    }
                    u = reduce(u, top16);
                    sc[0] = (int)f8_scale_byte<XF>(u << 16);
                    sc[1] = (int)f8_scale_byte<XF>(u & 0xffff0000u);
#pragma unroll
                    for (int q = 0; q < 8; ++q) xf[q] = (int)f8_cvt4_bf16<XF>(w[2 * q], w[2 * q + 1], f8_scale((unsigned)sc[q >> 2]));
                } else {
                    auto top32 = [](unsigned a, unsigned b) { return a > b ? a : b; };
                    float f[32];
                    if (whole) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) {                      // 32 floats; lanes behind K read zeros
                            const int col = c8 + 64 * (q >> 1 & 1) + 4 * (q & 1);
                            const uint4 v = load16(xbuf, col < a.K ? (row0 + (q >> 2)) * xpitch + 4 * col : (int)F8_OUTSIDE);
                            f[4 * q] = __uint_as_float(v.x); f[4 * q + 1] = __uint_as_float(v.y);
                            f[4 * q + 2] = __uint_as_float(v.z); f[4 * q + 3] = __uint_as_float(v.w);
                        }
                    } else {                                               // rows that start, or end, anywhere
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const long m = m0 + row0 + (q >> 1) < a.M ? m0 + row0 + (q >> 1) : a.M - 1;
                            const int col = c8 + 64 * (q & 1);
                            load8_tail<T>((const T*)a.x + (size_t)m * a.K + col, col, a.K, f + 8 * q);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        unsigned u = 0;
#pragma unroll
                        for (int e = 0; e < 16; ++e) u = top32(u, f8_mag(f[16 * h + e]));
                        sc[h] = (int)f8_scale_byte<XF>(reduce(u, top32));
                        const float inv = f8_inv_scale((unsigned)sc[h]);
#pragma unroll
                        for (int q = 4 * h; q < 4 * h + 4; ++q)
                            xf[q] = (int)f8_cvt4<XF>(f[4 * q] * inv, f[4 * q + 1] * inv, f[4 * q + 2] * inv, f[4 * q + 3] * inv);
                    }
                }
                xsc = odd ? sc[1] : sc[0];
                // after the swap xf[0 .. 3] are the even lane's pieces of this lane's row, xf[4 .. 7] the odd lane's
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    unsigned u = (unsigned)xf[q], w = (unsigned)xf[4 + q];
                    swap_pair(odd, u, w);
                    xf[q] = (int)u; xf[4 + q] = (int)w;
                }
                // xf[0,1], xf[4,5] are the halves of chunk g, xf[2,3], xf[6,7] those of chunk g + 4
                { const int t0 = xf[2], t1 = xf[3]; xf[2] = xf[4]; xf[3] = xf[5]; xf[4] = t0; xf[5] = t1; }
                if (a.q && n0 == 0 && 16 * i + r < mrem) {
                    const size_t row = (size_t)m0 + 16 * i + r;
                    uint4* to = reinterpret_cast<uint4*>(a.q + row * wp + c);
                    if (c < wp) to[0] = uint4{(unsigned)xf[0], (unsigned)xf[1], (unsigned)xf[2], (unsigned)xf[3]};
                    if (c + 64 < wp) to[4] = uint4{(unsigned)xf[4], (unsigned)xf[5], (unsigned)xf[6], (unsigned)xf[7]};
                    if (g == 0) {
                        a.scale[row * sp + kt] = (unsigned char)xsc;
                        for (int k = kt + 1; kt == kb - 1 && k < sp; ++k) a.scale[row * sp + k] = 127;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NF; ++j) block_product<XF, sizeof(TO) == 4>(acc[j][i], wf[j], xf, wsc[j], xsc);
        }
    }
#pragma unroll
    for (int half = NW / 2; half > 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int i = 0; i < MF; ++i) red[wave - half][j * MF + i][lane] = acc[j][i];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int i = 0; i < MF; ++i) acc[j][i] += red[wave][j * MF + i][lane];
        }
        __syncthreads();
    }
    // the last pair: wave 1 hands over, wave 0 stores
    if (wave == 1) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i) red[0][j * MF + i][lane] = acc[j][i];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i) store_quad<TO>(a, m0 + 16 * i + r, n0 + 16 * j + 4 * g, acc[j][i] + red[0][j * MF + i][lane]);
    }
}

// Tiled form, x packed: a workgroup of WM x WN waves owns BM rows x BN columns of y at a time.
//   K loop  = one block of 128 columns (128-byte rows of both operands) per step, two LDS stages filled by LDS-DMA one step
//             ahead.  A copy instruction moves 8 rows of 128 bytes.
//   tiles   = a workgroup walks its share of the tiles as one sequence of steps: the first step of the next tile is copied while
//             the last step of this one is multiplied, and the results are stored while it lands.
//   LDS     = 16-byte chunk c of row r lies at c ^ (r >> 1 & 7), and a lane takes chunks g and g + 4 of its row (g = lane / 16):
//             measured at 5.5 cycles per 1 KiB read with four waves reading, as fast as consecutive addresses; c ^ (r & 7), or
//             chunks 2g and 2g + 1, take 8.
//   scales  = the bytes of four steps are one dword per row, copied to LDS ahead of them as the operands are (loaded into
//             registers instead, the wait for them cost 15 % at K = 4096).
//   store   = lane pairs exchange quads (v_permlane16_swap), so that a lane writes eight consecutive columns of its row.
// Bound by the matrix units from K of about 1000 on: 16384 x 4096 -> 8192 462 us, 2380 TFLOP/s; below by HBM: 65536 x 384 -> 1152
// 47 us for 177 MB.
template <int BM, int BN> struct F8Tile {
    static constexpr int STAGE = (BM + BN) * F8_BLOCK;          // one step of both operands
    static constexpr int PANEL = BM * 4 + 256;                  // scales of four steps: BM rows, then the weight's row blocks
    static constexpr int LDS = 2 * STAGE + 2 * PANEL;
};

template <int XF, typename TO, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void linear_fp8_tile_kernel(F8LinArgs a) {
    using L = F8Tile<BM, BN>;
    constexpr int NW = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16;
    constexpr int STORES = MF * NF / 2 * (sizeof(TO) == 2 ? 1 : 2);       // of a wave and a whole tile
    // Copies are issued by one wave of each SIMD (CW of them): a wave sits in a copy's issue for longer than in a product's, and
    // meanwhile the SIMD's other wave multiplies (16384 x 4096 -> 8192: 489 us with all eight waves copying, 463 with four)
    constexpr int CW = NW == 8 ? 4 : NW;
    constexpr int XPW = BM / 8 / CW, WPW = BN / 8 / CW;                   // copy instructions per copying wave and step
    static_assert(CW % 2 == 0 && BM % (8 * CW) == 0 && BN % (8 * CW) == 0 && NF % 2 == 0 && MF % 4 == 0 && BN / WN <= F8_BLOCK && BM % 64 == 0 &&
                  BM <= 64 * NW, "tile");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int r = lane & 15, g = lane >> 4;
    const int kb = f8_blocks(a.K), pitch = f8_pitch(a.K), sp = f8_scale_pitch(a.K);

    // Order of the tiles: an XCD (workgroups id mod 8) takes a run of consecutive tiles, its workgroups in turn; the run goes
    // down 8 row tiles before along the columns, so that the tiles in flight on an XCD share rows of both operands.
    const int ntile = a.mtiles * a.ntiles, xcd = blockIdx.x & 7, nx = (gridDim.x + 7 - xcd) >> 3;
    const int q8 = ntile >> 3, r8 = ntile & 7;
    const int first = xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8;
    const int last = first + q8 + (xcd < r8 ? 1 : 0);

    const unsigned lds0 = lds_addr(smem);
    // In large tiles the products of widened operands (fp32 results) leave no registers for what copies and stores derive from the
    // lane: kept over the products it was spilled, and a reload waits for every copy before it.  There it is made anew, from a lane
    // number that the compiler knows nothing of, and a residual is loaded one row fragment at a time (us, before / after: 65536 x 128
    // -> 1024 76 / 56, with a residual 16384 x 4096 -> 8192 1171 / 1089, 32768 x 1024 -> 1024 142 / 110; small tiles, which have the
    // registers, lose 2 % by it).
    constexpr bool CROWDED = sizeof(TO) == 4 && BM > 128;
    auto fresh_lane = [&]() {
        int l = lane;
        if constexpr (CROWDED) asm volatile("" : "+v"(l));
        return l;
    };

    struct Tile { long m0; int n0; u32x4 x, w, xs, ws; };
    auto open = [&](int t) {
        const int per = 8 * a.ntiles, grp = t / per, in = t - grp * per;
        const int gm = a.mtiles - 8 * grp < 8 ? a.mtiles - 8 * grp : 8, col = in / gm;
        Tile o;
        // (divisions run on the vector unit: hand the results back to scalar registers)
        const int nt = __builtin_amdgcn_readfirstlane(col), mt = __builtin_amdgcn_readfirstlane(8 * grp + in - col * gm);
        o.m0 = (long)mt * BM; o.n0 = nt * BN;
        const int mrem = a.M - o.m0 < BM ? (int)(a.M - o.m0) : BM, nrem = a.N - o.n0 < BN ? a.N - o.n0 : BN;
        o.x = f8_buffer((const unsigned char*)a.x + (size_t)o.m0 * pitch, (unsigned)(mrem * pitch));
        o.w = f8_buffer(a.w + (size_t)o.n0 * pitch, (unsigned)(nrem * pitch));
        o.xs = f8_buffer(a.xs + (size_t)o.m0 * sp, (unsigned)(mrem * sp));
        o.ws = f8_buffer(a.ws + (size_t)(o.n0 / F8_BLOCK) * sp, (unsigned)(f8_blocks(nrem) * sp));
        return o;
    };
    // step kt of a tile into a stage, panel p of its scales into a slot
    auto stage = [&](const Tile& t, int kt, int buf) {
        // lane of a copy: row l/8 of its 8 rows, and the chunk that belongs at position l%8 of that row, if the row reaches that far
        const int l = fresh_lane(), lr = l >> 3, chunk = (l & 7) ^ ((4 * wave + (lr >> 1)) & 7);
        const unsigned off = kt * F8_BLOCK + 16 * chunk < pitch ? (unsigned)((8 * wave + lr) * pitch + 16 * chunk) : F8_OUTSIDE;
        const unsigned rowstep = (unsigned)(8 * CW * pitch), dst = lds0 + buf * L::STAGE + wave * 1024;
#pragma unroll
        for (int j = 0; j < XPW; ++j) buf_lds16(t.x, off + j * rowstep, kt * F8_BLOCK, dst + j * CW * 1024);
#pragma unroll
        for (int j = 0; j < WPW; ++j) buf_lds16(t.w, off + j * rowstep, kt * F8_BLOCK, dst + BM * F8_BLOCK + j * CW * 1024);
    };
    auto panel = [&](const Tile& t, int p, int slot) {
        const unsigned dst = lds0 + 2 * L::STAGE + slot * L::PANEL;
        const int l = fresh_lane();
        if (64 * wave < BM) buf_lds4(t.xs, (unsigned)((64 * wave + l) * sp), 4 * p, dst + wave * 256);
        if (wave == NW - 1) buf_lds4(t.ws, (unsigned)(l * sp), 4 * p, dst + BM * 4);
    };

    int t = first + (blockIdx.x >> 3);
    if (t >= last) return;
    Tile cur = open(t);
    int buf = 0, slot = 1;
    bool counted = false;
    panel(cur, 0, 0);
    if (wave < CW) stage(cur, 0, 0);

    // fragment addresses: row r of the wave's rows (rows 16 apart share their swizzle)
    const int c_lo = (g ^ (r >> 1)) << 4, c_hi = c_lo ^ 64;
    const int xrow = (wm * (BM / WM) + r) * F8_BLOCK, wrow = (BM + wn * (BN / WN) + r) * F8_BLOCK;
    const int wblock = wn * (BN / WN) / F8_BLOCK;

    for (;;) {
        f32x4 acc[MF][NF];
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int tn = t + nx;
        const bool more = tn < last;
        Tile nxt = cur;
        if (more) nxt = open(tn);
        for (int kt = 0; kt < kb; ++kt) {
            // the copies of this step are older than the stores of the tile before
            if (kt == 0 && counted) dma_wait_upto<STORES>(); else dma_wait_all();
            __syncthreads();               // this step is visible; every wave is done with the stage and slot refilled below
            const bool fin = kt + 1 == kb;
            if ((kt & 3) == 0) {
                slot ^= 1;
                if (kt + 4 < kb) panel(cur, (kt >> 2) + 1, slot ^ 1);
                else if (more) panel(nxt, 0, slot ^ 1);
            }
            if (wave < CW) {
                if (!fin) stage(cur, kt + 1, buf ^ 1);
                else if (more) stage(nxt, 0, buf ^ 1);
            }
            const unsigned char* st = smem + buf * L::STAGE;
            const unsigned char* scp = smem + 2 * L::STAGE + slot * L::PANEL + (kt & 3);
            const unsigned wsc = scp[BM * 4 + wblock * 4];
            unsigned xsc[MF];
#pragma unroll
            for (int i = 0; i < MF; ++i) xsc[i] = scp[(wm * (BM / WM) + 16 * i + r) * 4];
            i32x8 wf[NF];
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const unsigned char* p = st + wrow + j * 16 * F8_BLOCK;
                wf[j] = pair16(*reinterpret_cast<const uint4*>(p + c_lo), *reinterpret_cast<const uint4*>(p + c_hi));
            }
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                const unsigned char* p = st + xrow + i * 16 * F8_BLOCK;
                const i32x8 xf = pair16(*reinterpret_cast<const uint4*>(p + c_lo), *reinterpret_cast<const uint4*>(p + c_hi));
#pragma unroll
                for (int j = 0; j < NF; ++j) block_product<XF, sizeof(TO) == 4>(acc[i][j], wf[j], xf, (int)wsc, (int)xsc[i]);
            }
            buf ^= 1;
        }

        const int el = fresh_lane(), nb = cur.n0 + wn * (BN / WN) + (el >> 4 & 1) * 16 + (el >> 5) * 8;     // this lane's first column, pair 0
        float bias[NF / 2][8];
#pragma unroll
        for (int p = 0; p < NF / 2; ++p) {
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[p][e] = 0.0f;
            if (a.bias && nb + 32 * p < a.N) load8_tail<float>(a.bias + nb + 32 * p, nb + 32 * p, a.N, bias[p]);
        }
        auto piece = [&](int i, int p, float* v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][2 * p][e]),
                                                                 __float_as_uint(acc[i][2 * p + 1][e]), false, false);
                v[e] = __uint_as_float(sw[0]) + bias[p][e];
                v[4 + e] = __uint_as_float(sw[1]) + bias[p][4 + e];
            }
        };
        const long mb = cur.m0 + wm * (BM / WM) + r;
        // A whole tile is stored by straight code whose number of stores the next step's wait relies on; its residual is loaded
        // G row fragments at a time before their stores (a load behind a store waits for it: they complete in order).
        counted = cur.m0 + BM <= a.M && cur.n0 + BN <= a.N;
        if (counted) {
            constexpr int G = sizeof(TO) == 2 ? 4 : CROWDED ? 1 : 2;          // row fragments at a time: what registers hold
#pragma unroll
            for (int i0 = 0; i0 < MF; i0 += G) {
                Piece8<TO> res[G][NF / 2];
                if (a.residual) {
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int p = 0; p < NF / 2; ++p) res[i][p].load((const TO*)a.residual + (mb + 16 * (i0 + i)) * a.N + nb + 32 * p);
                }
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int p = 0; p < NF / 2; ++p) {
                        float v[8];
                        piece(i0 + i, p, v);
                        if (a.residual) res[i][p].add(v);
                        store8<TO>((TO*)a.y + (mb + 16 * (i0 + i)) * a.N + nb + 32 * p, v);
                    }
            }
        } else {
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int p = 0; p < NF / 2; ++p) {
                    float v[8];
                    piece(i, p, v);
                    const long m = mb + 16 * i;
                    const int n = nb + 32 * p;
                    if (m < a.M && n < a.N) {
                        if (a.residual) {
                            float f[8];
                            load8_tail<TO>((const TO*)a.residual + m * a.N + n, n, a.N, f);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] += f[e];
                        }
                        store8_tail<TO>((TO*)a.y + m * a.N + n, n, a.N, v);
                    }
                }
        }
        if (!more) break;
        t = tn;
        cur = nxt;
    }
}

// Row form: x in bf16 with rows of whole 16-byte pieces and at most nine blocks, many rows.  A workgroup of four waves (eight from
// five blocks on) rounds its 128 rows once, through LDS into the fragments' registers (and to memory, if the packed x is wanted),
// and then walks the columns in strips of 64, whose weights all waves read from LDS; LDS-DMA brings the next strip while one is
// multiplied and stored.  Bound by HBM: x is read once, where packing first writes and reads a byte more per element, in another
// launch.  65536 x 384 -> 384 25 us (100 MB, 4.0 TB/s), 32768 x 256 -> 768 21 us.
struct F8RowArgs {
    const bf16_t* x; const unsigned char* w; const unsigned char* ws; const float* bias; const bf16_t* residual; bf16_t* y;
    unsigned char* q; unsigned char* scale;        // the packed x, or null
    long M;
    int K, N, shares;                              // shares of the columns: workgroups that round the same rows
};

template <int KB, int NW>
__global__ __launch_bounds__(64 * NW, 2) void linear_fp8_rows_kernel(F8RowArgs a) {
    constexpr int ROWS = 128, MF = ROWS / 16 / NW, STRIP = 64 * KB * F8_BLOCK;      // rows of a workgroup, bytes of a strip
    constexpr int SD = (KB + 3) / 4;               // dwords of a row's scales
    static_assert(2 * STRIP == ROWS * KB * F8_BLOCK, "the strips take the place of the rounded rows");
    __shared__ __attribute__((aligned(16))) unsigned char xs[2 * STRIP];
    __shared__ unsigned sc[ROWS][SD];              // the rows' scales, a byte per block
    __shared__ __attribute__((aligned(16))) float extra[2][2][64];         // of a strip: its bias, and the scales of its weights
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const long mt = blockIdx.x / a.shares;
    const int share = (int)(blockIdx.x - mt * a.shares);
    const long m0 = mt * ROWS;
    const int mrem = a.M - m0 < ROWS ? (int)(a.M - m0) : ROWS;
    const int pitch = f8_pitch(a.K), sp = f8_scale_pitch(a.K);

    // ---- rounding: 16 lanes to a block, a pass of the workgroup is PASS rows
    {
        const int l = tid & 15, row0 = tid >> 4;
        const auto xbuf = f8_resource(a.x + (size_t)m0 * a.K, mrem * a.K * 2);
        const bool keep = a.q && share == 0;
        constexpr int PASS = 4 * NW, H = KB > 4 ? 2 : KB > 2 ? 4 : 8;      // H passes' loads are in flight together
#pragma unroll
        for (int h0 = 0; h0 < ROWS / PASS; h0 += H) {
            uint4 v[KB][H];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const int c = b * F8_BLOCK + 8 * l;
                    v[b][h] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                        xbuf, c < a.K ? ((row0 + PASS * (h0 + h)) * a.K + c) * 2 : (int)F8_OUTSIDE, 0, 0));
                }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int row = row0 + PASS * (h0 + h);
                unsigned scales[SD];
#pragma unroll
                for (int d = 0; d < SD; ++d) scales[d] = 0;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const unsigned* w = &v[b][h].x;
                    unsigned m = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned lo = w[e] & 0x7fffu, hi = w[e] >> 16 & 0x7fffu;
                        m = lo < 0x7f80u && lo > m ? lo : m;
                        m = hi < 0x7f80u && hi > m ? hi : m;
                    }
                    const unsigned s = f8_scale_byte<F8_E4M3>(row16_umax(m) << 16);
                    const float scale = f8_scale(s);
                    uint2 o;
                    o.x = f8_cvt4_bf16<F8_E4M3>(w[0], w[1], scale);
                    o.y = f8_cvt4_bf16<F8_E4M3>(w[2], w[3], scale);
                    *reinterpret_cast<uint2*>(xs + (b * ROWS + row) * F8_BLOCK + (((l >> 1) ^ (row >> 1 & 7)) << 4) + (l & 1) * 8) = o;
                    scales[b / 4] |= s << (8 * (b & 3));
                    if (keep && row < mrem && b * F8_BLOCK + 8 * l < pitch)
                        *reinterpret_cast<uint2*>(a.q + (size_t)(m0 + row) * pitch + b * F8_BLOCK + 8 * l) = o;
                }
#pragma unroll
                for (int b = KB; b < 4 * SD; ++b) scales[b / 4] |= 127u << (8 * (b & 3));
#pragma unroll
                for (int d = 0; d < SD; ++d) {
                    if (l == 0) sc[row][d] = scales[d];
                    if (keep && l == 0 && row < mrem) *reinterpret_cast<unsigned*>(a.scale + (size_t)(m0 + row) * sp + 4 * d) = scales[d];
                }
            }
        }
    }
    __syncthreads();

    // ---- this wave's rows as fragments: chunks g and g + 4 of row r, as in the tiled form
    i32x8 xf[KB][MF];
    unsigned xsc[MF][SD];
    const int c_lo = (g ^ (r >> 1)) << 4, c_hi = c_lo ^ 64;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
        for (int d = 0; d < SD; ++d) xsc[i][d] = sc[16 * (MF * wave + i) + r][d];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const unsigned char* p = xs + (b * ROWS + 16 * (MF * wave + i) + r) * F8_BLOCK;
            xf[b][i] = pair16(*reinterpret_cast<const uint4*>(p + c_lo), *reinterpret_cast<const uint4*>(p + c_hi));
        }
    }

    // ---- strips of 64 columns; this share's are a run of them.  In LDS: [block][64 rows of w][128 bytes]
    const int strips = (a.N + 63) / 64, per = (strips + a.shares - 1) / a.shares;
    const int first = share * per, end = first + per < strips ? first + per : strips;
    const int lr = lane >> 3, chunk = (lane & 7) ^ ((4 * wave + (lr >> 1)) & 7);
    const unsigned lds0 = lds_addr(xs), ex0 = lds_addr(extra);
    // A strip's groups of 8 rows, shared out to the waves block by block.  Only strips that exist: the scalar offset b * 128 is kept
    // below the buffer's size (a strip has a row at least), because the range check compares against size - scalar offset.
    auto load_strip = [&](int t, int buf) {
        const int nrem = a.N - 64 * t < 64 ? a.N - 64 * t : 64;
        const u32x4 wb = f8_buffer(a.w + (size_t)(64 * t) * pitch, (unsigned)(nrem * pitch));
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const unsigned off = b * F8_BLOCK + 16 * chunk < pitch ? (unsigned)((8 * wave + lr) * pitch + 16 * chunk) : F8_OUTSIDE;
#pragma unroll
            for (int j = 0; j < 8 / NW; ++j)
                buf_lds16(wb, off + j * 32 * pitch, b * F8_BLOCK, lds0 + buf * STRIP + b * 64 * F8_BLOCK + (4 * j + wave) * 1024);
        }
        // by LDS-DMA as well: the wait for an ordinary load would wait for the strip in front of it
        const u32x4 bb = f8_buffer((const unsigned char*)(a.bias + 64 * t), a.bias ? (unsigned)(nrem * 4) : 0u);
        if (wave == 2) buf_lds4(bb, lane * 4, 0, ex0 + buf * 512);
        if (wave == 3) buf_lds4(f8_buffer(a.ws + (size_t)(64 * t / F8_BLOCK) * sp, 4u * SD), lane * 4, 0, ex0 + buf * 512 + 256);
    };
    constexpr int STORES = MF * 2;
    __syncthreads();                               // every wave has its rows: the strips may take their place
    load_strip(first, 0);
    bool counted = false;
    for (int t = first; t < end; ++t) {
        const int buf = (t - first) & 1;
        if (counted) dma_wait_upto<STORES>(); else dma_wait_all();         // the strip is older than the stores of the one before
        __syncthreads();
        if (t + 1 < end) load_strip(t + 1, buf ^ 1);
        unsigned wsc[SD];
#pragma unroll
        for (int d = 0; d < SD; ++d) wsc[d] = __float_as_uint(extra[buf][1][d]);
        const int n = 64 * t + (g & 1) * 16 + (g >> 1) * 8;                 // this lane's first column when it stores, pair 0
        float bias[2][8];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4*>(&bias[p][e]) = *reinterpret_cast<const f32x4*>(&extra[buf][0][(n & 63) + 32 * p + e]);
        const bool whole = 64 * t + 64 <= a.N && mrem == ROWS;
        const long mb = m0 + 16 * MF * wave + r;
        Piece8<bf16_t> res[MF][2];
        if (a.residual && whole) {
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int p = 0; p < 2; ++p) res[i][p].load(a.residual + (mb + 16 * i) * a.N + n + 32 * p);
        }
        f32x4 acc[4][MF];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const unsigned char* st = xs + buf * STRIP + r * F8_BLOCK;
        auto wfrag = [&](int b, int j) {
            const unsigned char* p = st + (b * 64 + 16 * j) * F8_BLOCK;
            return pair16(*reinterpret_cast<const uint4*>(p + c_lo), *reinterpret_cast<const uint4*>(p + c_hi));
        };
#define BLOCK(b)                                                                                                                     \
    if constexpr (b < KB) {                                                                                                          \
        _Pragma("unroll") for (int j = 0; j < 4; ++j) {                                                                              \
            const i32x8 wf = wfrag(b, j);                                                                                            \
            _Pragma("unroll") for (int i = 0; i < MF; ++i) acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(             \
                wf, xf[b < KB ? b : 0][i], acc[j][i], F8_E4M3, F8_E4M3, b & 3, (int)wsc[b < KB ? b / 4 : 0], b & 3,                  \
                (int)xsc[i][b < KB ? b / 4 : 0]);                                                                                    \
        }                                                                                                                            \
    }
        BLOCK(0) BLOCK(1) BLOCK(2) BLOCK(3) BLOCK(4) BLOCK(5) BLOCK(6) BLOCK(7) BLOCK(8)
#undef BLOCK
        auto piece = [&](int i, int p, float* v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[2 * p][i][e]), __float_as_uint(acc[2 * p + 1][i][e]),
                                                                 false, false);
                v[e] = __uint_as_float(sw[0]) + bias[p][e];
                v[4 + e] = __uint_as_float(sw[1]) + bias[p][4 + e];
            }
        };
        counted = whole;
        if (whole) {
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[8];
                    piece(i, p, v);
                    if (a.residual) res[i][p].add(v);
                    store8<bf16_t>(a.y + (mb + 16 * i) * a.N + n + 32 * p, v);
                }
        } else {
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[8];
                    piece(i, p, v);
                    const int c = n + 32 * p;
                    if (mb + 16 * i < a.M && c < a.N) {
                        if (a.residual) {
                            float f[8];
                            load8_tail<bf16_t>(a.residual + (mb + 16 * i) * a.N + c, c, a.N, f);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] += f[e];
                        }
                        store8_tail<bf16_t>(a.y + (mb + 16 * i) * a.N + c, c, a.N, v);
                    }
                }
        }
    }
}

constexpr long LAUNCH_THREADS = 0xffffffffL;       // a launch counts fewer than 2^32 threads

template <int XK, int XF, typename TO, int MF, int NF, int NW> static int launch_direct(F8LinArgs a, hipStream_t s) {
    const long mtiles = (a.M + 16 * MF - 1) / (16 * MF);
    a.ntiles = (a.N + 16 * NF - 1) / (16 * NF);
    MAD_REQUIRE(mtiles * a.ntiles <= LAUNCH_THREADS / (64 * NW), "mad_linear_fp8: %ld rows x %d columns need more workgroups than a launch holds",
                a.M, a.N);
    hipLaunchKernelGGL((linear_fp8_direct_kernel<XK, XF, TO, MF, NF, NW>), dim3((unsigned)(mtiles * a.ntiles)), dim3(64 * NW), 0, s, a);
    return check_launch("mad_linear_fp8");
}

template <int XF, typename TO, int BM, int BN, int WM, int WN> static int launch_tile(F8LinArgs a, hipStream_t s) {
    constexpr int lds = F8Tile<BM, BN>::LDS, resident = 163840 / lds;
    const long mtiles = (a.M + BM - 1) / BM;
    a.ntiles = (a.N + BN - 1) / BN;
    MAD_REQUIRE(mtiles * a.ntiles <= 0x7fffffffL / 8, "mad_linear_fp8: %ld rows x %d columns need more tiles than the workgroups count",
                a.M, a.N);
    static int lds_dev = -1;
    auto kernel = &linear_fp8_tile_kernel<XF, TO, BM, BN, WM, WN>;
    MAD_REQUIRE(raise_lds_limit(reinterpret_cast<const void*>(kernel), lds, &lds_dev),
                "mad_linear_fp8: cannot raise the dynamic LDS limit to %d", lds);
    a.mtiles = (int)mtiles;
    const int tiles = a.mtiles * a.ntiles, grid = f8_cus() * resident;
    hipLaunchKernelGGL((linear_fp8_tile_kernel<XF, TO, BM, BN, WM, WN>), dim3(tiles < grid ? tiles : grid), dim3(64 * WM * WN), lds, s, a);
    return check_launch("mad_linear_fp8");
}

// Which form.  The units work in rounds of one tile of 256 x 256, or two of 128 x 128, each: the form whose rounds cover less area
// takes less time, where a round of small tiles counts 1.18 of its area from K = 1024 on (16384 x 4096 -> 4096 240 us with
// large tiles, 274 with small; 4096 x 4096 -> 1024 52 / 26) and nothing extra below (65536 x 384 -> 1152 51 / 47,
// 16384 x 256 -> 4096 37 / 37).  fp32 results, large / small: 8192 x 4096 -> 4096 239 / 271, 12288 x 2048 -> 6144 315 / 326,
// 65536 x 1152 -> 384 79 / 70, 65536 x 384 -> 1152 101 / 98, 16384 x 256 -> 4096 77 / 70.  With fewer than one small tile for each unit the direct form is as fast or faster
// (1024 x 4096 -> 1024 23 / 24, 64 x 256 -> 4096 3.5 / 5.7; fp32 777 x 1000 -> 328 7 / 15).
template <int XK, int XF, typename TO> static int launch_linear(F8LinArgs a, hipStream_t s) {
    if constexpr (XK < X_BF16) {
        const long cus = f8_cus(), small = ((a.M + 127) / 128) * ((a.N + 127) / 128), large = ((a.M + 255) / 256) * ((a.N + 255) / 256);
        if (small >= cus) {
            const long rl = (large + cus - 1) / cus * 4 * 100, rs = (small + 2 * cus - 1) / (2 * cus) * 2 * (a.K >= 1024 ? 118 : 100);
            return rl < rs ? launch_tile<XK, TO, 256, 256, 2, 4>(a, s) : launch_tile<XK, TO, 128, 128, 2, 2>(a, s);
        }
    }
    // Of the direct form, the smaller its workgroups the more of them share the latency, until re-reading costs more.  Sixteen by
    // sixteen results each up to two workgroups for each unit, then 32 x 32, then 64 x 64 (packed x, us, 16 / 32: 64 x 4096 -> 4096
    // 14.5 / 12.8, 256 x 4096 -> 1024 13.3 / 9.7; 32 / 64: 1024 x 4096 -> 1024 39 / 23).  Where x is rounded on its way in, every
    // workgroup rounds it again, so they get wider in n first (16 x 4096 -> 8192 10.6 / 8.2 for 16 / 32 columns), not in m, which
    // costs registers (32 x 4096 -> 8192 11.9 / 14.7 for 16 / 32 rows, fp32 777 x 1000 -> 328 9.6 / 12.3).  Eight waves, so that a
    // result is the same sum whether x came packed or is kept packed on the way (packed, four / eight waves in 32 x 32:
    // 1024 x 384 -> 384 4.4 / 4.7, fp32 64 x 4096 -> 4096 13.8 / 12.5).
    const long f = ((a.M + 15) / 16) * ((a.N + 15) / 16), cus = f8_cus();
    if constexpr (XK < X_BF16) {
        if (f <= 2 * cus) return launch_direct<XK, XF, TO, 1, 1, 8>(a, s);
        return f <= 8 * cus ? launch_direct<XK, XF, TO, 2, 2, 8>(a, s) : launch_direct<XK, XF, TO, 4, 4, 4>(a, s);
    } else {
        if (f <= cus) return launch_direct<XK, XF, TO, 1, 1, 8>(a, s);
        if (a.M <= 16 && !a.q) return launch_direct<XK, XF, TO, 1, 2, 16>(a, s);
        return launch_direct<XK, XF, TO, 1, 2, 8>(a, s);
    }
}

// Where the row form serves: bf16 rows of whole pieces, nine blocks at most (their fragments live in registers, two strips of the weights
// in LDS), rows enough for one workgroup to a unit, and no more columns than pay (us, packing first / rows: 32768 x 256 -> 768
// 27 / 21, 65536 x 384 -> 384 36 / 25, 32768 x 512 -> 2048 67 / 49, 40000 x 512 -> 4096 147 / 153, 65536 x 1152 -> 384 80 / 68,
// 32768 x 1024 -> 2048 94 / 84).  Beyond four blocks a unit holds one workgroup, and the last round has to be three quarters full
// (40000 x 640 -> 640 43 / 44, 40000 x 1152 -> 384 54 / 54).
static bool rows_form_ok(const void* x, int dtype, long rows, int K, int N) {
    const long tiles = (rows + 127) / 128, cus = f8_cus();
    return dtype == MAD_BF16 && whole_pieces(x, dtype, K) && K <= 9 * F8_BLOCK && N <= 2048 && tiles >= cus &&
           tiles <= LAUNCH_THREADS / 512 && (K <= 4 * F8_BLOCK || 4 * tiles >= 3 * ((tiles + cus - 1) / cus) * cus);
}

static F8RowArgs row_args(const void* x, const void* w, const void* ws, const float* bias, const void* residual, void* y, void* q,
                          void* scale, long rows, int K, int N) {
    F8RowArgs a;
    a.x = (const bf16_t*)x; a.w = (const unsigned char*)w; a.ws = (const unsigned char*)ws; a.bias = bias;
    a.residual = (const bf16_t*)residual; a.y = (bf16_t*)y; a.q = (unsigned char*)q; a.scale = (unsigned char*)scale;
    a.M = rows; a.K = K; a.N = N; a.shares = 1;
    return a;
}

static int launch_rows(F8RowArgs a, hipStream_t s) {
    const long mtiles = (a.M + 127) / 128;
    // with one workgroup to a unit its rounding, products and stores follow one another: two, of half the columns each, overlap
    // (32768 x 256 -> 768 25 us with one share, 22 with two); with more, rounding twice costs more (65536 x 384 -> 384 25 / 36)
    a.shares = a.K <= 4 * F8_BLOCK && mtiles < 2 * f8_cus() && a.N >= 256 ? 2 : 1;
    const dim3 grid((unsigned)(mtiles * a.shares));
#define ROWS(KB, NW) case KB: hipLaunchKernelGGL((linear_fp8_rows_kernel<KB, NW>), grid, dim3(64 * NW), 0, s, a); break
    switch (f8_blocks(a.K)) {
        ROWS(1, 4); ROWS(2, 4); ROWS(3, 4); ROWS(4, 4); ROWS(5, 8); ROWS(6, 8); ROWS(7, 8); ROWS(8, 8); ROWS(9, 8);
    }
#undef ROWS
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
    if (!packed && rows_form_ok(x, dtype, rows, K, N))
        return launch_rows(row_args(x, w, w_scale, bias, residual, y, nullptr, nullptr, rows, K, N), (hipStream_t)stream);
    F8LinArgs a;
    a.x = x; a.xs = (const unsigned char*)x_scale; a.w = (const unsigned char*)w; a.ws = (const unsigned char*)w_scale;
    a.q = a.scale = nullptr;
    a.bias = bias; a.residual = residual; a.y = y; a.M = rows; a.K = K; a.N = N; a.mtiles = a.ntiles = 0;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MAD_BF16) {
        if (x_type == MAD_E4M3) return launch_linear<X_E4M3, F8_E4M3, bf16_t>(a, s);
        if (x_type == MAD_E5M2) return launch_linear<X_E5M2, F8_E5M2, bf16_t>(a, s);
        return launch_linear<X_BF16, F8_E4M3, bf16_t>(a, s);
    }
    if (x_type == MAD_E4M3) return launch_linear<X_E4M3, F8_E4M3, float>(a, s);
    if (x_type == MAD_E5M2) return launch_linear<X_E5M2, F8_E5M2, float>(a, s);
    return launch_linear<X_F32, F8_E4M3, float>(a, s);
}

// Whether the direct form rounds x on its way in for less than a launch of its own costs: a few rows, or few 32 x 32 pieces of y and
// blocks for each (us of the GPU, rounding inside / packing first: bf16 777 x 1000 -> 328 7.0 / 8.8, 777 x 1000 -> 1024 13.1 / 12.4,
// 2048 x 1000 -> 1024 30 / 16, 256 x 4096 -> 1024 12.1 / 13.4, 256 x 4096 -> 4096 38 / 25; fp32, or rows that start anywhere, twice
// the work: fp32 777 x 1000 -> 328 8.8 / 8.8, 777 x 1000 -> 1024 17 / 13, 32 x 4096 -> 8192 18 / 12).  The host's time for the
// second launch and its buffers, 6 us, comes on top.
// Where the packed x is kept, only sizes whose packed form adds in the same order: y is then the product of what is kept, bit for bit.
static bool direct_rounds(const void* x, int dtype, long rows, int K, int N, bool keep) {
    const long cus = f8_cus(), wgs = ((rows + 31) / 32) * ((N + 31) / 32);
    if (keep && (((rows + 15) / 16) * ((N + 15) / 16) > 8 * cus || ((rows + 127) / 128) * ((N + 127) / 128) >= cus)) return false;
    const bool plain = dtype == MAD_BF16 && whole_pieces(x, dtype, K);
    return rows <= (plain ? 32 : 16) || (wgs <= 4 * cus && wgs * f8_blocks(K) * (plain ? 1 : 2) <= 32 * cus);
}

extern "C" int mad_linear_fp8_needs_pack(const void* x, int dtype, long rows, int K, int N) {
    return !direct_rounds(x, dtype, rows, K, N, false) && !rows_form_ok(x, dtype, rows, K, N);
}

extern "C" int mad_linear_fp8_save(const void* x, int dtype, int fmt, const void* w, const void* w_scale, const float* bias,
                                   const void* residual, void* y, void* q, void* scale, long rows, int K, int N, void* stream) {
    MAD_REQUIRE(rows >= 0 && N > 0 && N <= MAD_FP8_MAX_WIDTH, "mad_linear_fp8_save: bad shape rows=%ld N=%d", rows, N);
    const bool rows_form = fmt == MAD_E4M3 && K > 0 && rows_form_ok(x, dtype, rows, K, N);
    const bool typed = (dtype == MAD_BF16 || dtype == MAD_F32) && (fmt == MAD_E4M3 || fmt == MAD_E5M2);
    if (rows_form || (typed && rows > 0 && K > 0 && K <= MAD_FP8_MAX_WIDTH && direct_rounds(x, dtype, rows, K, N, true))) {
        MAD_REQUIRE(x && w && w_scale && y && q && scale, "mad_linear_fp8_save: null pointer");
        MAD_REQUIRE(f8_aligned(w, w_scale) && f8_aligned(q, scale),
                    "mad_linear_fp8_save: packed bytes must be 16-byte, scales 4-byte aligned");
        if (rows_form)
            return launch_rows(row_args(x, w, w_scale, bias, residual, y, q, scale, rows, K, N), (hipStream_t)stream);
        F8LinArgs a;
        a.x = x; a.xs = nullptr; a.w = (const unsigned char*)w; a.ws = (const unsigned char*)w_scale;
        a.q = (unsigned char*)q; a.scale = (unsigned char*)scale;
        a.bias = bias; a.residual = residual; a.y = y; a.M = rows; a.K = K; a.N = N; a.mtiles = a.ntiles = 0;
        hipStream_t s = (hipStream_t)stream;
        if (dtype == MAD_BF16)
            return fmt == MAD_E4M3 ? launch_linear<X_BF16, F8_E4M3, bf16_t>(a, s) : launch_linear<X_BF16, F8_E5M2, bf16_t>(a, s);
        return fmt == MAD_E4M3 ? launch_linear<X_F32, F8_E4M3, float>(a, s) : launch_linear<X_F32, F8_E5M2, float>(a, s);
    }
    if (int rc = mad_pack_fp8(x, dtype, fmt, rows, K, q, scale, stream)) return rc;
    return mad_linear_fp8(q, fmt, scale, w, w_scale, bias, residual, y, dtype, rows, K, N, stream);
}
