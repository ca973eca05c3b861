// hv_gemm_fp8.h -- Y = X8 . W8^T in OCP e4m3 with a scale for each block of 128 of the reduction, and the quantisation that
// makes the operands.
//
//   y[m][n] = bias[n] + residual[m][n] + sum_kb xs[m][kb] ws[n / 128][kb] sum_{k in block kb} x8[m][k] w8[n][k]
//
// A block of 128 is exactly one v_mfma_f32_16x16x128_f8f6f4: every instruction starts from a zero accumulator and its four
// results per lane are added to the fp32 sums with the block's factor xs ws -- 4 v_fma per 32-cycle MFMA, of which the matrix pipe hides a
// part (two waves a SIMD, 32 MFMAs and 128 v_fma a block in the order below: 539 ns, the MFMAs alone 462, the v_fma alone 128;
// profiles/operators_fp8_parts.txt).
// The operands are taken as A = W (rows n), B = X (columns m): a lane then owns ONE row m of Y per 16-row tile, so xs is one
// value per lane and tile, and the four W tiles of a 64-column block are read from LDS in an order that leaves the lane twice
// 8 consecutive columns: 16-byte stores, the four lanes of a row 64 bytes in one.
// Both operands are read with the same lane -> k assignment, so its order inside a block does not matter to the sum.
//
// Precision: the 8-bit matrix instructions (16x16x128 and 16x16x32 alike) add the products of 8 neighbouring k after aligning them
// to the largest of the eight with 13 bits kept behind it; the sums of those groups are exact to fp32 (measured, one product
// against another).  That is 1.6e-5 of the result (2-norm) for operands of like size, 5e-5 for operands over the whole e4m3 range:
// nothing to a bf16 output (1.7e-3), but an fp32 output would show it.  fp32 outputs are therefore computed on the bf16 instruction
// from the operands converted in registers (every e4m3 value is a bf16 value; its sums are exact to fp32: 8e-8 measured), at twice
// the matrix time.
#pragma once
#include "hv_common.h"
#include "humanvid_hip.h"

typedef int hv_i32x8 __attribute__((ext_vector_type(8)));  // 32 e4m3 values: the A / B operand of the 128-deep MFMA

HV_DEV f32x4 hv_mfma_fp8_128(hv_i32x8 a, hv_i32x8 b) {  // 16 x 16 x 128 from a zero accumulator
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#ifndef HV_EMU
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);  // e4m3 x e4m3, no hardware scale
#else
    return hvemu::mfma_fp8_128(a, b, zero);
#endif
}
// four floats -> four e4m3 (nearest, ties to even)
HV_DEV unsigned hv_e4m3x4(const float* f) {
#ifndef HV_EMU
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
#else
    return hvemu::cvt_pk_fp8(f[2], f[3], hvemu::cvt_pk_fp8(f[0], f[1], 0, false), true);
#endif
}
// 16 e4m3 values -> bf16, exactly
HV_DEV void hv_e4m3_to_bf16(u32x4 v, bf16x8* out) {
    u32x4 w[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#ifndef HV_EMU
        const unsigned lo = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.0f, false));
        const unsigned hi = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.0f, true));
#else
        auto two = [](unsigned b) { return hv_pack2(hvemu::fp8_to_f((unsigned char)b), hvemu::fp8_to_f((unsigned char)(b >> 8))); };
        const unsigned lo = two(v[i]), hi = two(v[i] >> 16);
#endif
        w[i / 2][2 * (i % 2)] = lo;
        w[i / 2][2 * (i % 2) + 1] = hi;
    }
    out[0] = hv_as_bf16x8(w[0]);
    out[1] = hv_as_bf16x8(w[1]);
}

// a lane's 32 values of one row and block, ready for the matrix instruction: as they are, or converted (WIDE: fp32 outputs)
template <bool WIDE>
struct HvFp8Frag {
    hv_i32x8 v;
    HV_DEV void set(u32x4 lo, u32x4 hi);
};
template <>
struct HvFp8Frag<true> {
    bf16x8 v[4];
    HV_DEV void set(u32x4 lo, u32x4 hi) {
        hv_e4m3_to_bf16(lo, v);
        hv_e4m3_to_bf16(hi, v + 2);
    }
};
HV_DEV hv_i32x8 hv_join32(u32x4 lo, u32x4 hi) {
    return hv_i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
template <>
HV_DEV void HvFp8Frag<false>::set(u32x4 lo, u32x4 hi) {
    v = hv_join32(lo, hi);
}
HV_DEV f32x4 hv_fp8_block_product(const HvFp8Frag<false>& a, const HvFp8Frag<false>& b) { return hv_mfma_fp8_128(a.v, b.v); }
HV_DEV f32x4 hv_fp8_block_product(const HvFp8Frag<true>& a, const HvFp8Frag<true>& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

struct HvGemmFp8Args {
    hv_gemm_fp8_params p;
    int kb;               // blocks of the reduction
    int tiles_m, tiles_n;
    int splits, per;      // ranges of the reduction (few tiles), blocks per range
};

// 16 bytes at any address of an element: rows of Y and the residual need not be aligned (129774 x 900 x 64: 77 us, 257 with single
// elements; 63515 x 1107 x 864 to fp32: 179 against 301)
HV_DEV u32x4 hv_ld16_any(const void* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <class V>
HV_DEV void hv_st16_any(void* p, V v) {
    static_assert(sizeof(V) == 16, "16 bytes");
    __builtin_memcpy(p, &v, 16);
}
// 8 consecutive columns n .. n + 7 of row m: residual, rounding, store
HV_DEV void hv_gemm_fp8_store(const HvGemmFp8Args& a, int m, int n, float* v) {
    const hv_gemm_fp8_params& p = a.p;
    if (n + 8 <= p.N) {
        if (p.residual) {
            float f[8];
            hv_unpack8(hv_ld16_any(p.residual + (long)m * p.ldr + n), f);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += f[i];
        }
        if (p.out_f32) {
            float* y = (float*)p.Y + (long)m * p.ldy + n;
            hv_st16_any(y, f32x4{v[0], v[1], v[2], v[3]});
            hv_st16_any(y + 4, f32x4{v[4], v[5], v[6], v[7]});
        } else {
            hv_st16_any((bf16_t*)p.Y + (long)m * p.ldy + n, hv_pack8(v));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (n + i < p.N) {
            float x = v[i];
            if (p.residual) x += hv_bf2f(p.residual[(long)m * p.ldr + n + i]);
            if (p.out_f32) ((float*)p.Y)[(long)m * p.ldy + n + i] = x;
            else ((bf16_t*)p.Y)[(long)m * p.ldy + n + i] = hv_f2bf(x);
        }
    }
}

// ---- tiles: WM x WN waves, a wave computes 16 MT rows x 64 columns; two LDS stages of one 128-block each, filled by LDS-DMA.
// LDS rows are 128 bytes (one block), their 16-byte pieces XOR-swizzled on the source side: X by (row >> 1) & 7; W, whose 16
// rows of an MFMA are 32 (i / 2) + 8 q + 4 (i & 1) + r, by (row >> 1 & 1) | (row >> 3 & 3) << 1 -- both leave the 16 lanes of a
// ds_read_b128 on 16 different quarters of the 64 banks.  The pieces behind K in the last block hold repeated values of the same row;
// their X side is zeroed in LDS.
// Workgroups are persistent: the first block of the next tile is on its way while the last one of this tile is computed and its
// results are stored -- one workgroup fills a CU's registers and LDS, so nothing else would cover that (147456 x 960 x 320: 124 us, 131 with
// a workgroup a tile).
// What bounds it, from builds that leave a part out (profiles/operators_fp8_parts.txt): 18432 x 10240 x 1280 takes 286 us (1690 TFLOP/s),
// 224 without the stores, 241 without the scales' multiply-adds, 236 without the copies, 183 without stores and multiply-adds.  The stores
// (377 MB) are the largest part that nothing covers.  Short reductions even more so: 147456 x 960 x 320 (283 MB of results) takes 121 us,
// 67 without the stores, 108 without the multiply-adds, 91 without the copies.  (The second block requested ahead of the stores too
// costs a barrier more and was slower: 138.)
// A whole tile's residual is requested four row tiles at a time (18432 x 10240 x 1280: 364 us, 407 when each row tile waits for its own;
// 147456 x 960 x 320: 181 and 191).
template <int WM, int WN, int MT, bool WIDE>
__global__ __launch_bounds__(64 * WM * WN, 2) void hv_gemm_fp8_kernel(HvGemmFp8Args a) {
    constexpr int BM = WM * MT * 16, BN = WN * 64, WAVES = WM * WN;
    constexpr int XB = BM * 128, WB = BN * 128, SB = BM * 4;       // bytes of a stage: X, W, the rows' scales
    constexpr int XI = XB / 1024 / WAVES, WI = WB / 1024 / WAVES;  // DMA instructions (1024 bytes) per wave and stage
    static_assert(XI * WAVES * 1024 == XB && WI * WAVES * 1024 == WB && BM / 64 <= WAVES && WAVES % 4 == 0, "whole instructions per wave");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * (XB + WB + SB)];
    __shared__ __attribute__((aligned(1024))) float sBias[2][BN];  // this tile's and the next one's
    const hv_gemm_fp8_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
#ifndef HV_EMU
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#else
    const int wave = tid >> 6;
#endif
    const int wm = wave % WM, wn = wave / WM;

    // an XCD takes a contiguous range of tiles, its workgroups the next ones in turn; inside it groups of 8 row tiles, the row tiles of a
    // column tile adjacent: the 32 tiles in flight share 8 panels of X and 4 of W in its L2
    const int total = a.tiles_m * a.tiles_n, per_xcd = (total + 7) / 8, turn = gridDim.x / 8;
    const int t_end = min(((int)(blockIdx.x & 7) + 1) * per_xcd, total);
    int t = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (t >= t_end) return;

    // DMA sources: instruction I = wave + WAVES i of a tile carries rows 8 I .. 8 I + 7, lane l the piece (l & 7) ^ key(row) of row
    // 8 I + l / 8; WAVES is a multiple of 4, so a lane's piece is the same for every i.  Rows past the end repeat the last row (their
    // products are never stored).
    const int xpiece = ((lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7)) * 16;
    const int wpiece = ((lane & 7) ^ (((lane >> 4) & 1) | ((wave & 3) << 1))) * 16;
    int m0 = 0, n0 = 0;
    const char *xbase = nullptr, *wbase = nullptr, *sbase = nullptr;
    const float* wsp = nullptr;
    unsigned xofs[XI], wofs[WI], sofs = 0;
    auto place = [&](int tile) {
        const int grp = tile / (8 * a.tiles_n), in_grp = tile % (8 * a.tiles_n), gm = min(8, a.tiles_m - grp * 8);
        m0 = (grp * 8 + in_grp % gm) * BM;
        n0 = in_grp / gm * BN;
        xbase = (const char*)p.X + (long)m0 * p.ldx;
        wbase = (const char*)p.W + (long)n0 * p.ldw;
        sbase = (const char*)(p.x_scale + (long)m0 * p.x_scale_row);
        wsp = p.w_scale + (long)(min(n0 + wn * 64, p.N - 1) / 128) * p.w_scale_row;
#pragma unroll
        for (int i = 0; i < XI; ++i) xofs[i] = (unsigned)min((wave + WAVES * i) * 8 + (lane >> 3), p.M - 1 - m0) * (unsigned)p.ldx;
#pragma unroll
        for (int i = 0; i < WI; ++i) wofs[i] = (unsigned)min((wave + WAVES * i) * 8 + (lane >> 3), p.N - 1 - n0) * (unsigned)p.ldw;
        if (wave < BM / 64) sofs = (unsigned)min(tid, p.M - 1 - m0) * (unsigned)(p.x_scale_row * 4);
    };
    float wnext = 0.f;
    auto issue = [&](int kb, int st) {
        unsigned char* xs = smem + st * (XB + WB + SB);
        unsigned char* ws = xs + XB;
        const int left = p.K - kb * 128 - 16;  // last piece inside K
        const unsigned xp = (unsigned)min(xpiece, left), wp = (unsigned)min(wpiece, left);
        wnext = wsp[(long)kb * p.w_scale_k];
#pragma unroll
        for (int i = 0; i < XI; ++i) hv_glds16_s(xbase + (long)kb * 128, xofs[i] + xp, xs + (wave + WAVES * i) * 1024);
#pragma unroll
        for (int i = 0; i < WI; ++i) hv_glds16_s(wbase + (long)kb * 128, wofs[i] + wp, ws + (wave + WAVES * i) * 1024);
        if (wave < BM / 64) hv_glds4_s(sbase + (long)kb * p.x_scale_k * 4, sofs, ws + WB + wave * 256);
    };
    auto issue_bias = [&](int which) {
        if (p.bias != nullptr && wave < BN / 64) hv_glds4_s(p.bias + n0, (unsigned)min(tid, p.N - 1 - n0) * 4u, &sBias[which][wave * 64]);
    };

    place(t);
    issue(0, 0);
    issue_bias(0);
    constexpr int SN = (WIDE ? 4 : 2) * MT;  // stores of a whole tile per lane
    bool stores = false;  // the last tile's SN stores, and nothing else, are younger than the copies in flight
    for (int st = 0, odd = 0;; odd ^= 1) {
        const int mt = m0, nt = n0;  // this tile
        const int next = t + turn;
        f32x4 acc[4][MT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int kb = 0; kb < a.kb; ++kb, st ^= 1) {
            if (kb == 0 && stores) hv_vm_wait<SN>();
            else hv_vm_wait<0>();
            hv_barrier_raw();  // block kb has landed, and nobody reads the other stage any more
            const float wsc = wnext;
            if (kb + 1 < a.kb) {
                issue(kb + 1, st ^ 1);
            } else if (next < t_end) {
                place(next);
                issue(0, st ^ 1);
                issue_bias(odd ^ 1);
            }
            unsigned char* xs = smem + st * (XB + WB + SB);
            const unsigned char* ws = xs + XB;
            const float* ss = reinterpret_cast<const float*>(ws + WB) + wm * MT * 16 + col;
            const int left = p.K - kb * 128;
            if (left < 128) {  // the last block is short: X is zero behind K
                for (int i = tid; i < BM * 8; i += 64 * WAVES) {
                    const int row = i >> 3;
                    if ((i & 7) * 16 >= left) hv_st16(xs + row * 128 + (((i & 7) ^ ((row >> 1) & 7)) << 4), u32x4{0u, 0u, 0u, 0u});
                }
                hv_barrier_raw();
            }
            // fragments: row 16 j + col of the wave's X rows, key (col >> 1); row 32 (i / 2) + 8 (col / 4) + 4 (i & 1) + col % 4 of its W rows
            const unsigned char* const xrow = xs + (wm * MT * 16 + col) * 128;
            const unsigned char* const wrow = ws + (wn * 64 + (col >> 2) * 8 + (col & 3)) * 128;
            const int xk = (g ^ (col >> 1)) << 4, wk = (g ^ (((col >> 1) & 1) | ((col >> 2) << 1))) << 4;  // the second piece: ^ 64
            HvFp8Frag<WIDE> wf[4], xf[2];
            f32x4 part[2][4];
            float f[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) wf[i].set(hv_ld16(wrow + (i / 2) * 4096 + (i & 1) * 512 + wk), hv_ld16(wrow + (i / 2) * 4096 + (i & 1) * 512 + (wk ^ 64)));
            xf[0].set(hv_ld16(xrow + xk), hv_ld16(xrow + (xk ^ 64)));
            f[0] = ss[0] * wsc;
            // row tile j's products are in flight while row tile j - 1's are added up
#pragma unroll
            for (int j = 0; j <= MT; ++j) {
                if (j + 1 < MT) xf[(j + 1) & 1].set(hv_ld16(xrow + (j + 1) * 2048 + xk), hv_ld16(xrow + (j + 1) * 2048 + (xk ^ 64)));
                if (j < MT) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[j & 1][i] = hv_fp8_block_product(wf[i], xf[j & 1]);
                }
                if (j > 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j - 1][r] = fmaf(part[(j - 1) & 1][i][r], f[(j - 1) & 1], acc[i][j - 1][r]);
                }
                if (j + 1 < MT) f[(j + 1) & 1] = ss[(j + 1) * 16] * wsc;
                hv_sched_fence();
            }
        }

        // a lane's results of row tile j: row mt + 16 (wm MT + j) + col, columns n .. n + 7 and n + 32 .. n + 39
        const int n = nt + wn * 64 + g * 8;
        float bias[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            f32x4 b = {0.f, 0.f, 0.f, 0.f};
            if (p.bias != nullptr) b = *reinterpret_cast<const f32x4*>(&sBias[odd][wn * 64 + g * 8 + (i / 8) * 32 + i % 8]);
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[i + e] = b[e];
        }
        stores = mt + BM <= p.M && nt + BN <= p.N;
        if (stores) {
            const long at = (long)(mt + wm * MT * 16 + col);
            char* y = (char*)p.Y + (at * p.ldy + n) * (WIDE ? 4 : 2);
            auto rows = [&](auto residual) {
                constexpr int RB = 4;  // row tiles whose residual is on its way at once
                const bf16_t* r = residual ? p.residual + at * p.ldr + n : nullptr;
#pragma unroll
                for (int jb = 0; jb < MT; jb += RB) {
                    u32x4 res[RB][2];
                    if (residual) {
#pragma unroll
                        for (int j = 0; j < RB; ++j, r += 16 * p.ldr) {
                            res[j][0] = hv_ld16_any(r);
                            res[j][1] = hv_ld16_any(r + 32);
                        }
                        hv_sched_fence();
                    }
#pragma unroll
                    for (int j = 0; j < RB; ++j, y += 16 * p.ldy * (WIDE ? 4 : 2)) {
                        float v[16], f[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = acc[i / 4][jb + j][i % 4] + bias[i];
                        if (residual) {
                            hv_unpack8(res[j][0], f);
                            hv_unpack8(res[j][1], f + 8);
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] += f[i];
                        }
                        if (WIDE) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) hv_st16_any(y + (i / 8 * 32 + i % 8) * 4, f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]});
                        } else {
                            hv_st16_any(y, hv_pack8(v));
                            hv_st16_any((bf16_t*)y + 32, hv_pack8(v + 8));
                        }
                    }
                }
            };
            if (p.residual) rows(std::true_type{});
            else rows(std::false_type{});
        } else {
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int m = mt + (wm * MT + j) * 16 + col;
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = acc[i / 4][j][i % 4] + bias[i];
                if (m < p.M) {
                    hv_gemm_fp8_store(a, m, n, v);
                    hv_gemm_fp8_store(a, m, n + 32, v + 8);
                }
            }
        }
        t = next;
        if (t >= t_end) break;
    }
}

// ---- few tiles: 64 x 64 of them, four waves of 16 rows, where 128 x 128 tiles would not give every CU one.  What counts there is the
// time a block of the reduction takes to arrive: four LDS stages, three blocks in flight, and with splits > 1 the blocks are divided among
// workgroups whose fp32 sums the join kernel adds up (in order: the result does not depend on which came first).  Every wave issues
// the same six copies a block (the scales four times over), so the waits can count them.
template <bool WIDE>
__global__ __launch_bounds__(256) void hv_gemm_fp8_small_kernel(HvGemmFp8Args a) {
    constexpr int XB = 64 * 128, STAGE = 2 * XB, S = 4;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[S * STAGE];
    __shared__ __attribute__((aligned(1024))) float sXs[S][64];
    __shared__ __attribute__((aligned(1024))) float sWs[S][64];
    const hv_gemm_fp8_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
#ifndef HV_EMU
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#else
    const int wave = tid >> 6;
#endif
    const int total = a.tiles_m * a.tiles_n, tile = blockIdx.x % total, split = blockIdx.x / total;
    const int m0 = tile % a.tiles_m * 64, n0 = tile / a.tiles_m * 64;
    const int k_begin = split * a.per, k_end = min(k_begin + a.per, a.kb);
    const char* const xbase = (const char*)p.X + (long)m0 * p.ldx;
    const char* const wbase = (const char*)p.W + (long)n0 * p.ldw;
    const int xpiece = ((lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7)) * 16;  // the tile kernel's swizzles
    const int wpiece = ((lane & 7) ^ (((lane >> 4) & 1) | ((wave & 3) << 1))) * 16;
    unsigned xofs[2], wofs[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        xofs[i] = (unsigned)min((wave + 4 * i) * 8 + (lane >> 3), p.M - 1 - m0) * (unsigned)p.ldx;
        wofs[i] = (unsigned)min((wave + 4 * i) * 8 + (lane >> 3), p.N - 1 - n0) * (unsigned)p.ldw;
    }
    const float* const sbase = p.x_scale + (long)m0 * p.x_scale_row;
    const unsigned sofs = (unsigned)min(lane, p.M - 1 - m0) * (unsigned)(p.x_scale_row * 4);
    const float* const wsp = p.w_scale + (long)(n0 / 128) * p.w_scale_row;  // 64 columns lie in one block of W's scales
    auto issue = [&](int kb) {
        const int st = kb & (S - 1);
        unsigned char* xs = smem + st * STAGE;
        const int left = p.K - kb * 128 - 16;
        const unsigned xp = (unsigned)min(xpiece, left), wp = (unsigned)min(wpiece, left);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            hv_glds16_s(xbase + (long)kb * 128, xofs[i] + xp, xs + (wave + 4 * i) * 1024);
            hv_glds16_s(wbase + (long)kb * 128, wofs[i] + wp, xs + XB + (wave + 4 * i) * 1024);
        }
        hv_glds4_s(sbase + (long)kb * p.x_scale_k, sofs, sXs[st]);
        hv_glds4_s(wsp + (long)kb * p.w_scale_k, 0u, sWs[st]);
    };
    f32x4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = k_begin; kb < min(k_begin + S - 1, k_end); ++kb) issue(kb);
    for (int kb = k_begin; kb < k_end; ++kb) {
        if (kb + 2 < k_end) hv_vm_wait<12>();  // two younger blocks may be in flight
        else if (kb + 1 < k_end) hv_vm_wait<6>();
        else hv_vm_wait<0>();
        hv_barrier_raw();  // block kb has landed, and nobody reads block kb - 1 any more
        if (kb + S - 1 < k_end) issue(kb + S - 1);
        unsigned char* const xs = smem + (kb & (S - 1)) * STAGE;
        const int left = p.K - kb * 128;
        if (left < 128) {
            for (int i = tid; i < 64 * 8; i += 256) {
                const int row = i >> 3;
                if ((i & 7) * 16 >= left) hv_st16(xs + row * 128 + (((i & 7) ^ ((row >> 1) & 7)) << 4), u32x4{0u, 0u, 0u, 0u});
            }
            hv_barrier_raw();
        }
        const unsigned char* const xrow = xs + (wave * 16 + col) * 128;
        const unsigned char* const wrow = xs + XB + ((col >> 2) * 8 + (col & 3)) * 128;
        const int xk = (g ^ (col >> 1)) << 4, wk = (g ^ (((col >> 1) & 1) | ((col >> 2) << 1))) << 4;
        HvFp8Frag<WIDE> wf[4], xf;
        xf.set(hv_ld16(xrow + xk), hv_ld16(xrow + (xk ^ 64)));
#pragma unroll
        for (int i = 0; i < 4; ++i) wf[i].set(hv_ld16(wrow + (i / 2) * 4096 + (i & 1) * 512 + wk), hv_ld16(wrow + (i / 2) * 4096 + (i & 1) * 512 + (wk ^ 64)));
        const float f = sXs[kb & (S - 1)][wave * 16 + col] * sWs[kb & (S - 1)][0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 part = hv_fp8_block_product(wf[i], xf);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(part[r], f, acc[i][r]);
        }
    }
    const int m = m0 + wave * 16 + col;
    if (m >= p.M) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = n0 + h * 32 + g * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[2 * h + i / 4][i % 4];
        if (a.splits > 1) {
            float* dst = p.workspace + ((long)split * p.M + m) * p.N + n;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n + i < p.N) dst[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += p.bias && n + i < p.N ? p.bias[n + i] : 0.f;
            hv_gemm_fp8_store(a, m, n, v);
        }
    }
}

__global__ __launch_bounds__(256) void hv_gemm_fp8_join_kernel(HvGemmFp8Args a) {
    const hv_gemm_fp8_params& p = a.p;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, all = (long)p.M * p.N;
    if (i >= all) return;
    const int m = (int)(i / p.N), n = (int)(i - (long)m * p.N);
    float v = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) v += p.workspace[(long)s * all + i];
    if (p.bias) v += p.bias[n];
    if (p.residual) v += hv_bf2f(p.residual[(long)m * p.ldr + n]);
    if (p.out_f32) ((float*)p.Y)[(long)m * p.ldy + n] = v;
    else ((bf16_t*)p.Y)[(long)m * p.ldy + n] = hv_f2bf(v);
}

// ---- few rows (M <= 16 MT): the weights' bytes are what counts.  A workgroup takes 16 columns; its eight waves take the blocks
// of the reduction in turn, operands straight from memory into registers a block ahead, and their sums are joined in LDS.
template <int MT, bool WIDE>
__global__ __launch_bounds__(512) void hv_gemm_fp8_rows_kernel(HvGemmFp8Args a) {
    __shared__ __attribute__((aligned(16))) float red[8][MT][64][4];
    const hv_gemm_fp8_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const unsigned char* wp = p.W + (long)min(n0 + col, p.N - 1) * p.ldw;
    const float* wsp = p.w_scale + (long)(n0 / 128) * p.w_scale_row;
    const unsigned char* xp[MT];
    const float* xsp[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = min(j * 16 + col, p.M - 1);
        xp[j] = p.X + (long)m * p.ldx;
        xsp[j] = p.x_scale + (long)m * p.x_scale_row;
        acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    struct Block {
        u32x4 w[2], x[MT][2];
        float f[MT];
    };
    auto load = [&](int kb) {  // what lies behind K is a repeated piece of W times zero
        Block b;
        const int k = kb * 128 + g * 32, k1 = min(k, p.K - 16), k2 = min(k + 16, p.K - 16);
        const u32x4 zero4 = {0u, 0u, 0u, 0u};
        b.w[0] = hv_ld16(wp + k1);
        b.w[1] = hv_ld16(wp + k2);
        const float wsc = wsp[(long)kb * p.w_scale_k];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            b.x[j][0] = k < p.K ? hv_ld16(xp[j] + k1) : zero4;
            b.x[j][1] = k + 16 < p.K ? hv_ld16(xp[j] + k2) : zero4;
            b.f[j] = xsp[j][(long)kb * p.x_scale_k] * wsc;
        }
        return b;
    };
    if (wave < a.kb) {
        Block next = load(wave);
        for (int kb = wave; kb < a.kb; kb += 8) {
            const Block b = next;
            if (kb + 8 < a.kb) next = load(kb + 8);
            HvFp8Frag<WIDE> wf;
            wf.set(b.w[0], b.w[1]);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                HvFp8Frag<WIDE> xf;
                xf.set(b.x[j][0], b.x[j][1]);
                const f32x4 part = hv_fp8_block_product(wf, xf);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(part[r], b.f[j], acc[j][r]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(red[wave][j][lane]) = acc[j];
    __syncthreads();
    for (int i = tid; i < MT * 256; i += 512) {
        const int j = i / 256, r = i % 16, c = i / 16 % 16;  // row m = 16 j + c, column n0 + r: neighbouring threads, neighbouring columns
        const int m = j * 16 + c, n = n0 + r;
        if (m >= p.M || n >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[w][j][(r / 4) * 16 + c][r % 4];
        if (p.bias) v += p.bias[n];
        if (p.residual) v += hv_bf2f(p.residual[(long)m * p.ldr + n]);
        if (p.out_f32) ((float*)p.Y)[(long)m * p.ldy + n] = v;
        else ((bf16_t*)p.Y)[(long)m * p.ldy + n] = hv_f2bf(v);
    }
}

static int g_hv_gemm_fp8_tile = 0;  // hv_set_tuning(HV_TUNE_GEMM_FP8)

// sizes -> kernel (its tile; 16: the rows kernel), tiles, ranges of the reduction; -1 invalid
static inline int hv_gemm_fp8_plan(const hv_gemm_fp8_params& p, HvGemmFp8Args& a, int& tile) {
    if (p.M < 0 || p.N < 0 || p.K < 16 || p.K % 16 != 0 || p.M > 0x7fffff00 || p.N > 0x7fffff00 || p.K > 0x7fffff00) return -1;
    a.p = p;
    a.kb = (p.K + 127) / 128;
    a.splits = 1;
    a.per = a.kb;
    a.tiles_m = a.tiles_n = 0;
    auto tiles = [&](int t) { return (long)((p.M + t - 1) / t) * ((p.N + t - 1) / t); };
    if (tiles(64) > 0x3fffffffL) return -1;
    const int want = g_hv_gemm_fp8_tile;
    // 256 tiles take 3.5 times a 128 tile's CU time and run one to a CU in whole rounds, 128 tiles two to a CU (K = 2560, 36864 x 640: 86 against
    // 73 us; 4096 x 4096 x 4096: 66 against 74); below 128 of the latter the 64 tiles' deeper pipeline and ranges are faster
    // (80 of them, 1024 x 1280 x 5120: 27 us, with 128 tiles 38; 160, 2048 x 1280 x 1280: 16 against 13).  An fp32 output's operands leave no room for 256.
    const long t256 = tiles(256), t128 = tiles(128);
    const bool large = !p.out_f32 && (t256 + 255) / 256 * 7 < 2 * (t128 < 512 ? 2 : (t128 + 255) / 256);
    tile = p.M <= 64 ? 16 : want ? (want == 256 && p.out_f32 ? 128 : want) : large ? 256 : t128 >= 128 ? 128 : 64;
    if (tile == 16) {
        a.tiles_m = 1;
        a.tiles_n = (p.N + 15) / 16;
        return hv_fits_launch(a.tiles_n, 512) ? 0 : -1;
    }
    a.tiles_m = (p.M + tile - 1) / tile;
    a.tiles_n = (p.N + tile - 1) / tile;
    if (tile == 64 && a.kb >= 16 && tiles(64) > 0 && tiles(64) <= 256) {  // ranges of at least 4 blocks: a join costs what 4 - 8 blocks do
        const long fill = 512 / tiles(64), most = a.kb / 4;
        a.splits = (int)(fill < most ? fill : most);
        a.per = (a.kb + a.splits - 1) / a.splits;
        a.splits = (a.kb + a.per - 1) / a.per;
    }
    if (tile == 64 && !hv_fits_launch(tiles(64) * a.splits, 256)) return -1;
    return 0;
}

static inline long hv_gemm_fp8_workspace_of(const hv_gemm_fp8_params& p) {
    HvGemmFp8Args a;
    int tile;
    if (hv_gemm_fp8_plan(p, a, tile) != 0) return -1;
    return a.splits > 1 ? (long)a.splits * p.M * p.N : 0;
}

static inline int hv_gemm_fp8_launch(const hv_gemm_fp8_params& p, hipStream_t stream) {
    HvGemmFp8Args a;
    int tile;
    if (hv_gemm_fp8_plan(p, a, tile) != 0) return -1;
    if (p.ldx % 16 != 0 || p.ldw % 16 != 0 || (((uint64_t)p.X | (uint64_t)p.W) & 15) != 0) return -1;
    if (p.ldx < 0 || p.ldw < 0 || p.ldx > (1L << 23) || p.ldw > (1L << 23)) return -1;  // 256 rows within 32-bit offsets
    if (p.x_scale_row < 0 || p.x_scale_row > (1L << 21) || (p.M > 1 && p.ldy < p.N) || p.ldr < 0) return -1;
    if (p.M == 0 || p.N == 0) return 0;
    const long floats = a.splits > 1 ? (long)a.splits * p.M * p.N : 0;
    if (floats > p.workspace_floats || (floats > 0 && (p.workspace == nullptr || ((uint64_t)p.workspace & 3) != 0))) return -3;
    const long total = (long)a.tiles_m * a.tiles_n, turns = (total + 7) / 8 * 8;
    hv_note("hv_gemm_fp8_kernel %d | M=%d N=%d K=%d ranges=%d", tile, p.M, p.N, p.K, a.splits);
    auto go = [&](auto wide) {
        constexpr bool WIDE = decltype(wide)::value;
        if (tile == 16) {
            const dim3 grid((unsigned)a.tiles_n), block(512);
            if (p.M <= 16) hv_launch(hv_gemm_fp8_rows_kernel<1, WIDE>, grid, block, stream, a);
            else if (p.M <= 32) hv_launch(hv_gemm_fp8_rows_kernel<2, WIDE>, grid, block, stream, a);
            else hv_launch(hv_gemm_fp8_rows_kernel<4, WIDE>, grid, block, stream, a);
        } else if (tile == 256) {
            hv_launch(hv_gemm_fp8_kernel<2, 4, 8, false>, dim3((unsigned)(turns < 256 ? turns : 256)), dim3(512), stream, a);
        } else if (tile == 128) {
            hv_launch(hv_gemm_fp8_kernel<2, 2, 4, WIDE>, dim3((unsigned)(turns < 512 ? turns : 512)), dim3(256), stream, a);
        } else {
            hv_launch(hv_gemm_fp8_small_kernel<WIDE>, dim3((unsigned)(total * a.splits)), dim3(256), stream, a);
        }
    };
    if (p.out_f32) go(std::true_type{});
    else go(std::false_type{});
    if (a.splits > 1) {
        hv_note("hv_gemm_fp8_join_kernel | M=%d N=%d ranges=%d", p.M, p.N, a.splits);
        hv_launch(hv_gemm_fp8_join_kernel, dim3((unsigned)(((long)p.M * p.N + 255) / 256)), dim3(256), stream, a);
    }
    return 0;
}

// ---- quantisation to e4m3 with a scale for each 1 x 128 (block_rows 1: activations) or 128 x 128 block (weights) -----------------
//   s = max(max|x| / 448, 2^-126), 1 for a block of zeros;  q = the e4m3 value nearest to x 448 / max|x| (ties to even).
// The quotient of two bf16 numbers often lies exactly between two e4m3 values, and x * (448 / max|x|) in fp32 may miss such a
// middle by its rounding (2^-23).  x 448 / max|x| is a quotient of integers below 2^11 and 2^8: it is on a middle (at most 5
// significant bits) or at least 2^-13 away from it, relatively.  Rounding the product to 16 significant bits before the
// conversion therefore gives the conversion of the exact quotient.
HV_DEV float hv_row16_max(float x) {
#ifndef HV_EMU
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 0xf, 0xf, true)));
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 0xf, 0xf, true)));
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xf, 0xf, true)));
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x140, 0xf, 0xf, true)));
#else
    for (int o = 1; o < 16; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
#endif
    return x;
}
HV_DEV float hv_amax8(u32x4 v) {  // max |x| of 8 bf16 (a NaN is passed over: it does not set a scale)
    float f[8];
    hv_unpack8(v, f);
    float m = fabsf(f[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
    return fmaxf(m, 0.f);
}
HV_DEV float hv_fp8_block_scale(float amax, float& inv) {
    const float s = amax / 448.0f;
    if (amax == 0.f) {
        inv = 1.f;
        return 1.f;
    }
    if (s < 1.17549435e-38f) {  // 2^-126, the smallest normal number
        inv = 8.50705917e37f;   // 2^126
        return 1.17549435e-38f;
    }
    inv = 448.0f / amax;
    return s;
}
HV_DEV u32x2 hv_quant8(u32x4 v, float inv) {
    float f[8];
    hv_unpack8(v, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = __builtin_bit_cast(uint32_t, f[e] * inv);
        f[e] = __builtin_bit_cast(float, (u + 0x80u) & ~0xffu);
    }
    return u32x2{hv_e4m3x4(f), hv_e4m3x4(f + 4)};
}

struct HvQuantArgs {
    const bf16_t* X;
    unsigned char* Q;
    float* scale;
    long ldx, ldq, scale_row, scale_k;
    int M, K, kb;
};

// one scale per row and block: 16 lanes per (row, block), 16 bytes per lane
__global__ __launch_bounds__(256) void hv_fp8_quantize_rows_kernel(HvQuantArgs a) {
    const int lane16 = threadIdx.x & 15;
    const long items = (long)a.M * a.kb;
    const long i = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool live = i < items;  // no early return: every lane takes part in the reduction below
    const long row = live ? i / a.kb : 0;
    const int blk = live ? (int)(i % a.kb) : 0;
    const int k = blk * 128 + lane16 * 8;
    const bool on = live && k < a.K;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (on) v = hv_ld16(a.X + row * a.ldx + k);
    const float amax = hv_row16_max(hv_amax8(v));
    float inv;
    const float s = hv_fp8_block_scale(amax, inv);
    if (on) hv_st8(a.Q + row * a.ldq + k, hv_quant8(v, inv));
    if (live && lane16 == 0) a.scale[row * a.scale_row + (long)blk * a.scale_k] = s;
}

// one scale per 128 x 128 block: a workgroup holds the block in registers
__global__ __launch_bounds__(256) void hv_fp8_quantize_blocks_kernel(HvQuantArgs a) {
    __shared__ float top[4];
    const int tid = threadIdx.x, blk = blockIdx.x, m0 = blockIdx.y * 128;
    const int k = blk * 128 + (tid & 15) * 8;
    u32x4 v[8];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = m0 + i * 16 + (tid >> 4);
        v[i] = u32x4{0u, 0u, 0u, 0u};
        if (row < a.M && k < a.K) v[i] = hv_ld16(a.X + (long)row * a.ldx + k);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, hv_amax8(v[i]));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if ((tid & 63) == 0) top[tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    float inv;
    const float s = hv_fp8_block_scale(amax, inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = m0 + i * 16 + (tid >> 4);
        if (row < a.M && k < a.K) hv_st8(a.Q + (long)row * a.ldq + k, hv_quant8(v[i], inv));
    }
    if (tid == 0) a.scale[(long)blockIdx.y * a.scale_row + (long)blk * a.scale_k] = s;
}

static inline int hv_fp8_quantize_launch(const HvQuantArgs& in, int block_rows, hipStream_t stream) {
    HvQuantArgs a = in;
    if (a.M < 0 || a.K <= 0 || a.K % 16 != 0 || a.K > 0x7fffff00 || a.M > 0x7fffff00 || a.ldx % 8 != 0 || a.ldq % 16 != 0) return -1;
    if ((block_rows != 1 && block_rows != 128) || (a.M > 1 && (a.ldq < a.K || a.ldx < 0))) return -1;
    if ((((uint64_t)a.X | (uint64_t)a.Q) & 15) != 0) return -1;
    if (a.M == 0) return 0;
    a.kb = (a.K + 127) / 128;
    if (block_rows == 1) {
        const long wgs = ((long)a.M * a.kb + 15) / 16;
        if (!hv_fits_launch(wgs, 256)) return -1;
        hv_note("hv_fp8_quantize_rows_kernel | M=%d K=%d", a.M, a.K);
        hv_launch(hv_fp8_quantize_rows_kernel, dim3((unsigned)wgs), dim3(256), stream, a);
    } else {
        if ((a.M + 127) / 128 > 65535) return -1;
        hv_note("hv_fp8_quantize_blocks_kernel | M=%d K=%d", a.M, a.K);
        hv_launch(hv_fp8_quantize_blocks_kernel, dim3((unsigned)a.kb, (unsigned)((a.M + 127) / 128)), dim3(256), stream, a);
    }
    return 0;
}
