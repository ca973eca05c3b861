// hv_cross_attention.h -- attention of Lq queries to an encoder's Lk states (Lk of any length, unrelated to Lq), with a key
// mask, attended lengths and shared key heads.  The UNets' attn2 with more than one encoder token
// (/root/reference/src/models/attention.py:410-424, diffusers Attention with encoder_hidden_states).
//
//   s[i][j] = scale * q[i] . k[j],  p = softmax over the attended j,  o[i] = sum_j p[i][j] v[j]      (0 where nothing is attended)
//
// One pass over the states with the running maximum m and sum l of the softmax: a chunk of CH = 32 NP keys contributes
//   m' = max(m, max_j s),  p_j = 2^((s_j - m') scale log2 e),  (l, o) = (l, o) 2^((m - m') scale log2 e) + sum_j p_j (1, v_j).
// m, l and o are fp32; p is rounded to bf16 for the second product (2^-8 relative, the operands' own precision), and l sums
// those rounded p (a product with a row of ones), so that the weights of a row add up to one exactly.
//
// Layout: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16.  A lane owns one query column (lane & 15) and 4 of every 16
// key rows ((lane >> 4) * 4 + r): the maximum needs two lane-swap steps per chunk, and the p of two 16-key tiles ARE the B
// operand of the second product if its reduction index runs over the keys in that order (k = 8 g + e is key 4 g + e of the
// first tile for e < 4, of the second for e >= 4); V is stored row-major in LDS and read transposed in the same order.
// A masked key's row of K and V is zero in LDS (whatever memory holds there) and its score starts at -inf: the accumulator of
// the first product is initialised with the chunk's bias (0 / -inf) instead of zero, so masks cost no instruction.  (A query that holds
// NaN or infinity makes such a score NaN and spoils its row, as its attended states' scores do anyway.  Chunks without an attended
// state are passed over, so that an entry without any gives zeros whatever its queries hold.)
// Query heads that share a key head are rows of the same tile: row r of a (batch, key head) is query r / G, head r % G.
#pragma once
#include "hv_common.h"
#include "humanvid_hip.h"

// a NaN wins (v_maximum3_f32: no quieting of the operands first, as fmaxf would have it): its row is NaN either way
HV_DEV float hv_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
HV_DEV float hv_max5(float m, const f32x4& s) { return hv_max(hv_max(hv_max(hv_max(m, s[0]), s[1]), s[2]), s[3]); }

#ifndef HV_EMU
// max over the four lanes with equal lane & 15
HV_DEV float hv_max_quarters(float x) {
    // (the halves are copied out first: a bit cast of a vector element takes element 0)
    unsigned u = __builtin_bit_cast(unsigned, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // a[0]: the lower half's values in both halves, a[1]: the upper's
    unsigned lo = a[0], hi = a[1];
    x = hv_max(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
    u = __builtin_bit_cast(unsigned, x);
    const auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);  // the same for the two 16-lane rows of a half
    lo = b[0], hi = b[1];
    return hv_max(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
#else
HV_DEV float hv_max_quarters(float x) {
    x = hv_max(x, __shfl_xor(x, 32));
    return hv_max(x, __shfl_xor(x, 16));
}
#endif

struct HvCrossArgs {
    hv_cross_attention_params p;
    float c;             // scale * log2 e
    int G, rows;         // heads per key head; rows of a (batch, key head): Lq * G
    int kernel;          // 0: few states, 1: few rows, 2: any, one 16-row tile per wave, 3: any, two
    int blocks;          // row blocks of a (batch, key head); few states: tiles of queries
    int per_wg, groups;  // few states: tiles one workgroup takes, workgroups per entry and head group
    int splits, per;     // ranges the keys are cut into, keys per range
    int run;             // neighbouring units that go to one XCD
    int units;           // workgroups with work
};

#define HV_CROSS_FEW_ROWS(D) ((D) == 40 ? 64 : 32)  // hv_cross_attention_few_kernel: queries whose pieces fill whole copy instructions

// row r of a (batch, key head) is query r / G, head r % G of the key head's G
HV_DEV void hv_cross_row(const HvCrossArgs& a, int r, int kvh, int& query, int& column) {
    if (a.G == 1) {  // (uniform: spares the division)
        query = r;
        column = kvh * a.p.D;
    } else {
        query = r / a.G;
        column = (kvh * a.G + (r - query * a.G)) * a.p.D;
    }
}

// workspace of a call whose keys are cut into ranges: per (batch, key head, row, range) D unnormalised sums, and behind all of those
// the maximum and the sum of weights they refer to
HV_DEV float* hv_cross_weights(const HvCrossArgs& a) {
    return a.p.workspace + (long)a.p.B * a.p.kv_heads * a.rows * a.splits * a.p.D;
}

// geometry of the LDS copies and of a lane's share of the output for head dim D
template <int D>
struct HvCrossGeom {
    static constexpr int KS = (D + 31) / 32, DT = (D + 15) / 16, P8 = D / 8;
    static constexpr int KSTR = KS * 64 + 16;                 // bytes of a K row: an odd number of 16-byte pieces (no bank conflicts)
    static constexpr int VSTR = (DT % 2 ? DT : DT + 1) * 32;  // bytes of a V row: an odd number of 32-byte tiles (the transposed reads)
    // output tiles come in pairs that share 32 columns: row 4 c + r of the first is column 8 c + r, of the second 8 c + 4 + r, so that a
    // lane's eight values are neighbours (16-byte stores); an odd last tile is in order
    static constexpr int PAIRED = DT / 2 * 2;
    HV_DEV static int vbyte(int dt, int c) { return dt < PAIRED ? dt / 2 * 64 + c * 16 + (dt & 1) * 8 : dt * 32 + c * 8; }
};

// A operand of O^T = V^T P^T for output tile dt and the 32 keys from row0 on: lane t of a 16-lane group points at row t / 4, column
// group t % 4 and receives column t of the 4 rows; the second read takes the 16-key tile behind
template <int D>
HV_DEV bf16x8 hv_cross_vfrag(const unsigned char* sV, int row0, int dt, int col, int g) {
    using G = HvCrossGeom<D>;
    const unsigned char* src = sV + (row0 + g * 4 + col / 4) * G::VSTR + G::vbyte(dt, col & 3);
    const bf16x4 v0 = hv_lds_tr4(src), v1 = hv_lds_tr4(src + 16 * G::VSTR);
    return bf16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
}

// a row's D values of a head: o = acc / sum of weights, 0 where that is 0 (nothing attended); at(piece) is where its 16-byte piece lies
template <int D, class At>
HV_DEV void hv_cross_store(At at, const f32x4* acc, float sum, int g) {
    using G = HvCrossGeom<D>;
    const float inv = sum == 0.f ? 0.f : __builtin_amdgcn_rcpf(sum);  // (within 2^-23: the output keeps 2^-8)
#pragma unroll
    for (int d = 0; d < G::PAIRED; d += 2)
        hv_st16(at(d * 2 + g), u32x4{hv_pack2(acc[d][0] * inv, acc[d][1] * inv), hv_pack2(acc[d][2] * inv, acc[d][3] * inv),
                                     hv_pack2(acc[d + 1][0] * inv, acc[d + 1][1] * inv), hv_pack2(acc[d + 1][2] * inv, acc[d + 1][3] * inv)});
    if constexpr (G::DT % 2 == 1) {
        constexpr int d = G::DT - 1;
        if (d * 16 + g * 4 < D)
            hv_st8((char*)at(d * 2 + g / 2) + (g & 1) * 8, u32x2{hv_pack2(acc[d][0] * inv, acc[d][1] * inv), hv_pack2(acc[d][2] * inv, acc[d][3] * inv)});
    }
}

#ifndef HV_EMU
HV_DEV unsigned long hv_ballot(bool x) { return __ballot(x); }
#else
HV_DEV unsigned long hv_ballot(bool x) {
    unsigned long r = 0;
    for (int i = 0; i < 64; ++i) r |= (unsigned long)(__shfl((int)x, i) != 0) << i;
    return r;
}
#endif

// between a wave's own LDS writes and other lanes' reads of them: the LDS serves a wave in order, the compiler has to keep that order
HV_DEV void hv_wave_fence() {
#ifndef HV_EMU
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#else
    (void)__shfl_xor(0, 1);  // the emulator runs lanes one after the other up to the next collective
#endif
}

HV_DEV bf16x8 hv_bf16_ones() { return bf16x8{0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80}; }

// ---- few states (Lk <= 16 NT <= 96, D <= 80): a prompt.  The stream of queries is what counts -- q is read once, o written once.
// A workgroup takes four neighbouring query heads (4 / G key heads) and streams tiles of TQ queries through two LDS slots: the next
// tile is in flight by LDS-DMA while this one is computed, the results replace the queries in the slot and leave it.  Both ways a
// row's four heads are one run of memory (320 - 640 bytes).  At 2 x 147456 queries, 77 states, D = 40 (378 MB) it takes 90 - 96 us; a head
// at a time took 115, straight from memory into operand registers (16 lanes in 16 rows) 133.
// All of K and V^T of its key head stay in a wave's REGISTERS as matrix operands.  No running maximum: a row's scores are all there.
// The number of 16-key tiles is a template argument: branches around absent tiles cost more than a masked tile.  2, 4, 5 and 6 tiles are
// there: 1 and 3 would spare little beside the stream of queries (16 states as one tile or two: 83.4 against 83.8 us at D = 40,
// 32.4 against 32.8 at D = 80; 33 states as three or four: 86.9 against 87.8 and 35.1 against 36.2).
template <int D, int NT>
__global__ __launch_bounds__(256, D == 40 ? 3 : 2) void hv_cross_attention_few_kernel(HvCrossArgs a) {
    using G = HvCrossGeom<D>;
    constexpr int KS = G::KS, DT = G::DT, P8 = G::P8, NP = (NT + 1) / 2, CH = 32 * NP;
    constexpr int TQ = HV_CROSS_FEW_ROWS(D), NPC = 4 * P8, NI = TQ * NPC / 256, SLOT = TQ * NPC * 16;
    static_assert(TQ * NPC % 256 == 0, "whole copy instructions per wave");
    constexpr int VPART = 32 * G::VSTR;  // a wave's 32 rows of V, before the slots are used
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * SLOT > 4 * VPART ? 2 * SLOT : 4 * VPART];
    __shared__ __attribute__((aligned(16))) float sBias[CH];
    const int per_xcd = (a.units + 7) / 8;  // neighbouring units (the head groups of one range of rows) on one XCD
    const int unit = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || unit >= a.units) return;
    const hv_cross_attention_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
#ifndef HV_EMU
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#else
    const int wave = tid >> 6;
#endif
    const int hgroups = p.heads / 4, hgroup = unit % hgroups, group = unit / hgroups % a.groups, b = unit / hgroups / a.groups;
    const int kvh = (hgroup * 4 + wave) / a.G;
    int len = p.kv_len ? p.kv_len[b] : p.Lk;
    len = len < 0 ? 0 : len > p.Lk ? p.Lk : len;
    const u32x4 zero4 = {0u, 0u, 0u, 0u};
    bf16x8 kf[NT][KS], vf[NP][DT];
    {
        const bf16_t* Kb = p.K + (long)b * p.k_stride_b + (long)kvh * D;
        const bf16_t* Vb = p.V + (long)b * p.v_stride_b + (long)kvh * D;
        const uint8_t* mask = p.key_mask ? p.key_mask + (long)b * p.mask_stride_b : nullptr;
        unsigned char* const part = smem + wave * VPART;
        constexpr int VP = DT * 2;  // pieces of a padded V row
        bool some = false;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            const int row = kt * 16 + col;
            const bool on = row < len && (mask == nullptr || mask[row] != 0);
            some = some || on;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                kf[kt][ks] = hv_as_bf16x8(on && ks * 32 + g * 8 < D ? hv_ld16(Kb + (long)row * p.ldk + ks * 32 + g * 8) : zero4);
        }
        if (hv_ballot(some) == 0) {  // (the same in all four waves) nothing attended: zeros, the queries are not looked at
            const int q0 = group * a.per_wg * TQ, queries = min(a.per_wg * TQ, p.Lq - q0);
            bf16_t* const O = p.O + (long)b * p.o_stride_b + (long)q0 * p.ldo + (long)hgroup * 4 * D;
            for (long i = tid; i < (long)queries * NPC; i += 256) hv_st16(O + i / NPC * p.ldo + i % NPC * 8, zero4);
            return;
        }
#pragma unroll
        for (int pr = 0; pr < NP; ++pr) {
            for (int i = lane; i < 32 * VP; i += 64) {
                const int row = pr * 32 + i / VP, piece = i % VP;
                const bool on = row < len && piece < P8 && (mask == nullptr || mask[row] != 0);
                hv_st16(part + i / VP * G::VSTR + piece * 16, on ? hv_ld16(Vb + (long)row * p.ldv + piece * 8) : zero4);
            }
            hv_wave_fence();
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[pr][d] = hv_cross_vfrag<D>(part, 0, d, col, g);
            hv_wave_fence();
        }
        if (tid < CH) sBias[tid] = tid < len && (mask == nullptr || mask[tid] != 0) ? 0.f : -INFINITY;
    }
    hv_barrier_raw();  // every wave has its operands (the barrier waits for LDS reads): copies may land in the slots

    // slot layout: query-major, NPC 16-byte pieces a query (its four heads), rotated by a function of the query so that the 16 rows of a
    // fragment access lie in 16 different quarters of the banks: NPC = 20, 32, 40 repeat after 4, 1, 2 queries
    constexpr int SH = NPC % 32 == 0 ? 0 : NPC % 8 == 0 ? 1 : 2;
    auto rotated = [](int query, int piece) {
        const int at = piece + ((query >> SH) & (15 >> SH));
        return at < NPC ? at : at - NPC;
    };
    const bf16_t* const Qb = p.Q + (long)b * p.q_stride_b + (long)hgroup * 4 * D;
    bf16_t* const Ob = p.O + (long)b * p.o_stride_b + (long)hgroup * 4 * D;
    auto offset = [&](int i, int last, long ld) {  // byte offset inside a tile of the piece that lane and instruction i carry
        const int idx = (wave * NI + i) * 64 + lane, slot = idx % NPC, query = idx / NPC;
        int piece = slot - ((query >> SH) & (15 >> SH));
        piece = piece < 0 ? piece + NPC : piece;
        return (unsigned)min(query, last) * (unsigned)(ld * 2) + (unsigned)(piece * 16);
    };
    unsigned qofs[NI], oofs[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        qofs[i] = offset(i, TQ, p.ldq);
        oofs[i] = offset(i, TQ, p.ldo);
    }
    unsigned char* slot = smem;
    unsigned char* other = smem + SLOT;
    auto issue = [&](int tile, unsigned char* to) {
        const char* base = (const char*)(Qb + (long)tile * TQ * p.ldq);
        const int last = p.Lq - 1 - tile * TQ;
        if (last >= TQ - 1) {
#pragma unroll
            for (int i = 0; i < NI; ++i) hv_glds16_s(base, qofs[i], to + (wave * NI + i) * 1024);
        } else {  // queries behind the last repeat it and are not stored
#pragma unroll
            for (int i = 0; i < NI; ++i) hv_glds16_s(base, offset(i, last, p.ldq), to + (wave * NI + i) * 1024);
        }
    };
    // rows of this wave: the G query heads of its key head are G waves' rows, TQ each; row r = wave's share * TQ + i of them is query
    // r / G, head r % G
    const int share = wave % a.G;
    const int end = min((group + 1) * a.per_wg, a.blocks);  // tiles of TQ queries
    int tile = group * a.per_wg;
    issue(tile, slot);
    for (bool first = true; tile < end; ++tile, first = false) {
        // in flight, in order: this tile's copies, the stores of the tile before (all NI of them: it was not the last)
        if (first) hv_vm_wait<0>();
        else hv_vm_wait<NI>();
        hv_barrier_raw();  // the tile is there, and nobody reads the other slot any more
        if (tile + 1 < end) issue(tile + 1, other);
#pragma unroll 1
        for (int sub = 0; sub < TQ; sub += 16) {
            int query = sub + col, head = wave;
            if (a.G > 1) {  // (uniform)
                const int r = share * TQ + query;
                query = r / a.G;
                head = wave - share + r % a.G;
            }
            unsigned char* const row = slot + query * (NPC * 16);
            f32x4 s[NT];
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) s[kt] = *reinterpret_cast<const f32x4*>(sBias + kt * 16 + g * 4);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 q = zero4;
                if ((ks + 1) * 32 <= D || ks * 32 + g * 8 < D) q = hv_ld16(row + rotated(query, head * P8 + ks * 4 + g) * 16);
#pragma unroll
                for (int kt = 0; kt < NT; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt][ks], hv_as_bf16x8(q), s[kt], 0, 0, 0);
            }
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) top = hv_max5(top, s[kt]);
            top = hv_max_quarters(top);
            const float mc = top == -INFINITY ? 0.f : -top * a.c;  // nothing attended: 2^(-inf - 0) = 0
            f32x4 acc[DT], sum;
#pragma unroll
            for (int pr = 0; pr < NP; ++pr) {
                u32x4 w = zero4;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (2 * pr + h < NT) {
                        float f[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = __builtin_amdgcn_exp2f(fmaf(s[2 * pr + h][e], a.c, mc));
                        w[2 * h] = hv_pack2(f[0], f[1]);
                        w[2 * h + 1] = hv_pack2(f[2], f[3]);
                    }
                const bf16x8 pf = hv_as_bf16x8(w);
                const f32x4 none = {0.f, 0.f, 0.f, 0.f};
                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_bf16_ones(), pf, pr ? sum : none, 0, 0, 0);
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[pr][d], pf, pr ? acc[d] : none, 0, 0, 0);
            }
            // (the pieces of these rows and heads are this wave's alone, and it has read them)
            hv_wave_fence();
            hv_cross_store<D>([&](int piece) { return row + rotated(query, head * P8 + piece) * 16; }, acc, sum[0], g);
        }
        hv_barrier_raw();  // the results of all four waves are in the slot
        char* base = (char*)(Ob + (long)tile * TQ * p.ldo);
        u32x4 out[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) out[i] = hv_ld16(slot + (wave * NI + i) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (tile * TQ + ((wave * NI + i) * 64 + lane) / NPC < p.Lq) hv_st16(base + oofs[i], out[i]);
        unsigned char* const t = slot;
        slot = other;
        other = t;
    }
}

// which part of the work a workgroup of the kernels below takes.  The states of a (batch, key head) are read by all of its row
// blocks and should stay in one L2: neighbouring units (row blocks of the same keys, in runs of a.run) go to one XCD, the runs to the
// XCDs in turn, so that entries of different lengths spread over all of them.  The keys are cut into ranges of a.per keys
// whatever an entry's length: workgroups are equally long, those behind an entry's end leave at once.
struct HvCrossPart {
    int b, kvh, block, split, begin, end;
    bool none;
};
HV_DEV HvCrossPart hv_cross_part(const HvCrossArgs& a) {
    const hv_cross_attention_params& p = a.p;
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    const int run = (at / a.run) * 8 + xcd, unit = run * a.run + at % a.run;
    HvCrossPart w;
    w.none = unit >= a.units;
    w.block = unit % a.blocks;
    int rest = unit / a.blocks;
    w.split = rest % a.splits;
    rest /= a.splits;
    w.kvh = rest % p.kv_heads;
    w.b = w.none ? 0 : rest / p.kv_heads;
    int len = p.kv_len ? p.kv_len[w.b] : p.Lk;
    len = len < 0 ? 0 : len > p.Lk ? p.Lk : len;
    w.begin = min(w.split * a.per, len);
    w.end = min(w.begin + a.per, len);
    w.none = w.none || (w.split > 0 && w.begin >= w.end);  // (the join does not read it; range 0 is always there)
    return w;
}

// The running maximum is moved only where a score passes it by more than 2^8: the weights then stay below 2^8, their sums far inside
// fp32, and the products by 2^((m - m') c) are rare after the first chunk.
#define HV_CROSS_SLACK 8.0f

// ---- any number of states: a workgroup's 64 QT rows go through the keys in chunks of CH, two LDS stages filled by LDS-DMA, one
// barrier a chunk.  Rows of K and V lie in LDS as in memory (D values), their 16-byte pieces rotated by a function of the row
// so that the 16 rows of an access lie in different banks (5, 8, 10, 16 or 20 pieces a row repeat the banks after 16, 2, 8, 1, 4 rows).
// In a chunk with a mask, or behind the end, the rows that are not attended are zeroed first.
template <int D>
struct HvCrossChunk {
    static constexpr int P8 = D / 8, CH = D >= 128 ? 32 : 64, T = P8 % 16 == 0 ? 4 : P8 % 8 == 0 ? 3 : P8 % 4 == 0 ? 2 : P8 % 2 == 0 ? 1 : 0;
    static constexpr int TILE = CH * D * 2, STAGE = 2 * TILE;
    HV_DEV static int rot(int row) { return (row >> (4 - T)) & ((1 << T) - 1); }
    HV_DEV static int at(int row, int piece) {  // byte offset of a piece
        const int slot = piece + rot(row);
        return (row * P8 + (slot < P8 ? slot : slot - P8)) * 16;
    }
};
template <int D, int QT>
__global__ __launch_bounds__(256, QT == 1 && D < 128 ? 3 : 2) void hv_cross_attention_kernel(HvCrossArgs a) {
    using Geom = HvCrossGeom<D>;
    using Chunk = HvCrossChunk<D>;
    constexpr int KS = Geom::KS, DT = Geom::DT, P8 = Geom::P8, CH = Chunk::CH, KT = CH / 16;
    constexpr int CI = CH * P8 / 64, NI = (2 * CI + 3) / 4;  // copy instructions of a K or V tile; of both, per wave
    static_assert(CH * P8 % 64 == 0, "whole copy instructions");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * Chunk::STAGE];
    __shared__ __attribute__((aligned(16))) float sBias[3][CH];  // zeros, and one for each stage
    const HvCrossPart part = hv_cross_part(a);
    if (part.none) return;
    const hv_cross_attention_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
#ifndef HV_EMU
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#else
    const int wave = tid >> 6;
#endif
    const int b = part.b, kvh = part.kvh;
    const int chunks = (part.end - part.begin + CH - 1) / CH;
    const bf16_t* const Kb = p.K + (long)b * p.k_stride_b + (long)kvh * D;
    const bf16_t* const Vb = p.V + (long)b * p.v_stride_b + (long)kvh * D;
    const uint8_t* const mask = p.key_mask ? p.key_mask + (long)b * p.mask_stride_b : nullptr;
    const u32x4 zero4 = {0u, 0u, 0u, 0u};

    // copy instruction j = wave + 4 i: pieces 64 j .. of the K tile, behind CI those of the V tile
    auto offset = [&](int j, int last) {
        const int idx = (j < CI ? j : j - CI) * 64 + lane, row = idx / P8, slot = idx % P8;
        int piece = slot - Chunk::rot(row);
        piece = piece < 0 ? piece + P8 : piece;
        return (unsigned)min(row, last) * (unsigned)((j < CI ? p.ldk : p.ldv) * 2) + (unsigned)(piece * 16);
    };
    unsigned ofs[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) ofs[i] = offset(wave + 4 * i, CH);
    uint8_t keep_next = 1;  // this lane's key of the next chunk
    auto issue = [&](int ch, unsigned char* stage) {
        const int k0 = part.begin + ch * CH, last = part.end - 1 - k0;
        const char* const kb = (const char*)(Kb + (long)k0 * p.ldk);
        const char* const vb = (const char*)(Vb + (long)k0 * p.ldv);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int j = wave + 4 * i;
            if (j < 2 * CI) hv_glds16_s(j < CI ? kb : vb, last >= CH - 1 ? ofs[i] : offset(j, last), stage + j * 1024);
        }
        if (mask != nullptr) keep_next = lane <= last && lane < CH ? mask[k0 + lane] : 0;
    };
    if (chunks > 0) issue(0, smem);
    if (tid < CH) sBias[0][tid] = 0.f;

    const int r0 = (part.block * 4 + wave) * QT * 16 + col;
    bf16x8 qf[QT][KS];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = r0 + t * 16;
        int query, column;
        hv_cross_row(a, r, kvh, query, column);
        const bf16_t* src = p.Q + (long)b * p.q_stride_b + (long)query * p.ldq + column;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qf[t][ks] = hv_as_bf16x8(r < a.rows && ks * 32 + g * 8 < D ? hv_ld16(src + ks * 32 + g * 8) : zero4);
    }
    int kat[KS], vat[(DT + 1) / 2];  // a lane's places in the K tile (its row col) and in the V tile (row 4 g + col / 4)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kat[ks] = Chunk::at(col, ks * 4 + g);
#pragma unroll
    for (int d = 0; d < (DT + 1) / 2; ++d)
        vat[d] = Chunk::TILE + (2 * d < Geom::PAIRED ? Chunk::at(g * 4 + col / 4, d * 4 + (col & 3)) : Chunk::at(g * 4 + col / 4, d * 4 + (col & 3) / 2) + (col & 1) * 8);

    f32x4 acc[QT][DT], lsum[QT];
    float m[QT], mc[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = -INFINITY;
        mc[t] = 0.f;
        lsum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int ch = 0; ch < chunks; ++ch) {
        unsigned char* const stage = smem + (ch & 1) * Chunk::STAGE;
        const int n = part.end - part.begin - ch * CH;
        hv_vm_wait<0>();
        hv_barrier_raw();  // the chunk has landed, and nobody reads the other stage any more
        const bool kept = keep_next != 0;
        if (ch + 1 < chunks) issue(ch + 1, smem + ((ch + 1) & 1) * Chunk::STAGE);
        const float* bias = sBias[0] + g * 4;  // zeros
        if (mask != nullptr || n < CH) {
            const unsigned long keep = hv_ballot(lane < CH && lane < n && kept);
            for (int i = tid; i < 2 * CH * P8; i += 256) {  // (rows keep their place: any order of the pieces will do)
                const int row = i % CH, piece = i / CH;
                if (!(keep >> row & 1ul)) hv_st16(stage + (piece < P8 ? 0 : Chunk::TILE) + (row * P8 + (piece < P8 ? piece : piece - P8)) * 16, zero4);
            }
            bias = sBias[1 + (ch & 1)] + g * 4;
            if (tid < CH) sBias[1 + (ch & 1)][tid] = keep >> tid & 1ul ? 0.f : -INFINITY;
            hv_barrier_raw();
            if (keep == 0) continue;  // (the same in all four waves)
        }
        f32x4 s[QT][KT];
        u32x4 kv[2][KS];  // the next 16 keys' operands are read while this 16's are used; fences keep it at that
        auto read_k = [&](int kt) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kv[kt & 1][ks] = zero4;
                if ((ks + 1) * 32 <= D || ks * 32 + g * 8 < D) kv[kt & 1][ks] = hv_ld16(stage + kat[ks] + kt * (16 * P8 * 16));
            }
        };
        read_k(0);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            if (kt + 1 < KT) read_k(kt + 1);
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t][kt] = *reinterpret_cast<const f32x4*>(bias + kt * 16);
            if (kt < 2 || n > 32) {  // (a last chunk of at most 32 keys leaves its second half out)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int t = 0; t < QT; ++t)
                        s[t][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_as_bf16x8(kv[kt & 1][ks]), qf[t][ks], s[t][kt], 0, 0, 0);
            }
            hv_sched_fence();
        }
        bf16x4 v0[2], v1[2];  // V fragments, one output tile ahead
        auto read_v = [&](int i) {
            const int pr = i / DT, d = i % DT;
            const unsigned char* src = stage + vat[d / 2] + (d < Geom::PAIRED ? (d & 1) * 8 : 0) + pr * (32 * P8 * 16);
            v0[i & 1] = hv_lds_tr4(src);
            v1[i & 1] = hv_lds_tr4(src + 16 * P8 * 16);
        };
        read_v(0);
        float top[QT];
        bool past = false;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            top[t] = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) top[t] = hv_max5(top[t], s[t][kt]);
            top[t] = hv_max_quarters(top[t]);
            past = past || (top[t] - m[t]) * a.c > HV_CROSS_SLACK;
        }
        if (__any(past)) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float mn = hv_max(m[t], top[t]);
                const float ms = mn == -INFINITY ? 0.f : mn;  // nothing attended yet: 2^(-inf - 0) = 0, not 2^(-inf + inf)
                const float alpha = __builtin_amdgcn_exp2f((m[t] - ms) * a.c);
                m[t] = mn;
                mc[t] = -ms * a.c;
#pragma unroll
                for (int e = 0; e < 4; ++e) lsum[t][e] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][d][e] *= alpha;
            }
        }
#pragma unroll
        for (int pr = 0; pr < KT / 2; ++pr) {
            if (pr > 0 && n <= 32) break;
            bf16x8 pf[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __builtin_amdgcn_exp2f(fmaf(s[t][2 * pr + e / 4][e % 4], a.c, mc[t]));
                pf[t] = hv_as_bf16x8(hv_pack8(f));
            }
#pragma unroll
            for (int t = 0; t < QT; ++t) lsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_bf16_ones(), pf[t], lsum[t], 0, 0, 0);
            hv_sched_fence();
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int i = pr * DT + d;
                if (i + 1 < DT * KT / 2) read_v(i + 1);
                const bf16x4 x = v0[i & 1], y = v1[i & 1];
                const bf16x8 vf = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
                for (int t = 0; t < QT; ++t) acc[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[t], acc[t][d], 0, 0, 0);
                hv_sched_fence();
            }
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = r0 + t * 16;
        if (r >= a.rows) continue;
        if (a.splits > 1) {  // unnormalised sums, with the maximum and the sum of weights they refer to
            const long at = (((long)b * p.kv_heads + kvh) * a.rows + r) * a.splits + part.split;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int c = d < Geom::PAIRED ? d / 2 * 32 + g * 8 + (d & 1) * 4 : d * 16 + g * 4;
                if (c < D) *reinterpret_cast<f32x4*>(p.workspace + at * D + c) = acc[t][d];
            }
            if (g == 0) *reinterpret_cast<f32x2*>(hv_cross_weights(a) + at * 2) = f32x2{m[t], lsum[t][0]};
        } else {
            int query, column;
            hv_cross_row(a, r, kvh, query, column);
            bf16_t* dst = p.O + (long)b * p.o_stride_b + (long)query * p.ldo + column;
            hv_cross_store<D>([&](int piece) { return dst + piece * 8; }, acc[t], lsum[t][0], g);
        }
    }
}

// ---- at most 16 rows (Lq G <= 16): reading the states is all there is.  The four waves of a workgroup take blocks of 32 keys in turn,
// each on its own: K straight from memory into operand registers, V through 32 rows of LDS of its own (for the transposed read), both
// requested a block ahead -- 16 KB in flight per wave at D = 128, and no barrier until the four results are joined in LDS.
template <int D>
__global__ __launch_bounds__(256, 2) void hv_cross_attention_rows_kernel(HvCrossArgs a) {
    using Geom = HvCrossGeom<D>;
    constexpr int KS = Geom::KS, DT = Geom::DT, P8 = Geom::P8, VSTR = Geom::VSTR;
    constexpr int NV = (32 * P8 + 63) / 64;  // 16-byte pieces of V per lane and block
    constexpr int VPART = 32 * VSTR, JOIN = 16 * (D + 2) * 4;
    constexpr int OWN = VPART > JOIN ? VPART : JOIN;
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * OWN];
    const HvCrossPart part = hv_cross_part(a);
    if (part.none) return;
    const hv_cross_attention_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int b = part.b, kvh = part.kvh;
    const bf16_t* Kb = p.K + (long)b * p.k_stride_b + (long)kvh * D;
    const bf16_t* Vb = p.V + (long)b * p.v_stride_b + (long)kvh * D;
    const uint8_t* mask = p.key_mask ? p.key_mask + (long)b * p.mask_stride_b : nullptr;
    unsigned char* const sV = smem + wave * OWN;
    const u32x4 zero4 = {0u, 0u, 0u, 0u};
    if constexpr (DT * 2 > P8) {
        if (lane < 32) hv_st16(sV + lane * VSTR + P8 * 16, zero4);
    }
    bf16x8 qf[KS];
    {
        int query, column;
        hv_cross_row(a, col, kvh, query, column);
        const bf16_t* src = p.Q + (long)b * p.q_stride_b + (long)query * p.ldq + column;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qf[ks] = hv_as_bf16x8(col < a.rows && ks * 32 + g * 8 < D ? hv_ld16(src + ks * 32 + g * 8) : zero4);
    }
    f32x4 acc[DT], lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, mc = 0.f;
    u32x4 kreg[2][KS], vreg[NV];
    bool on[2] = {false, false};  // whether this lane's key of a 16-key tile (its col) is attended
    auto fetch = [&](int k0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row = k0 + t * 16 + col;
            on[t] = row < part.end && (mask == nullptr || mask[row] != 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                kreg[t][ks] = row < part.end && ks * 32 + g * 8 < D ? hv_ld16(Kb + (long)row * p.ldk + ks * 32 + g * 8) : zero4;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = i * 64 + lane, row = k0 + idx / P8;
            vreg[i] = idx < 32 * P8 && row < part.end ? hv_ld16(Vb + (long)row * p.ldv + idx % P8 * 8) : zero4;
        }
    };
    int k0 = part.begin + wave * 32;
    if (k0 < part.end) fetch(k0);
    for (; k0 < part.end; k0 += 128) {
        // bit j: key k0 + j is attended (lanes 0 - 15 hold the tile's keys)
        unsigned keep = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) keep |= (unsigned)(hv_ballot(on[t]) & 0xffffu) << (16 * t);
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = keep >> (t * 16 + g * 4 + e) & 1u ? 0.f : -INFINITY;
            if (keep == 0) continue;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_as_bf16x8(on[t] ? kreg[t][ks] : zero4), qf[ks], s[t], 0, 0, 0);
        }
        hv_wave_fence();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = i * 64 + lane, row = idx / P8;
            if (idx < 32 * P8) hv_st16(sV + row * VSTR + idx % P8 * 16, keep >> row & 1u ? vreg[i] : zero4);
        }
        hv_wave_fence();
        if (k0 + 128 < part.end) fetch(k0 + 128);
        float top = hv_max_quarters(hv_max5(hv_max5(-INFINITY, s[0]), s[1]));
        if (__any((top - m) * a.c > HV_CROSS_SLACK)) {
            const float mn = hv_max(m, top), ms = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f((m - ms) * a.c);
            m = mn;
            mc = -ms * a.c;
#pragma unroll
            for (int e = 0; e < 4; ++e) lsum[e] *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[d][e] *= alpha;
        }
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __builtin_amdgcn_exp2f(fmaf(s[e / 4][e % 4], a.c, mc));
        const bf16x8 pf = hv_as_bf16x8(hv_pack8(f));
        lsum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_bf16_ones(), pf, lsum, 0, 0, 0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hv_cross_vfrag<D>(sV, 0, d, col, g), pf, acc[d], 0, 0, 0);
    }
    // the four waves' results: [wave][row][m, l, D sums]
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(smem) + (wave * 16 + col) * (D + 2);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int at = d < Geom::PAIRED ? d / 2 * 32 + g * 8 + (d & 1) * 4 : d * 16 + g * 4;
        if (at < D) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[2 + at + e] = acc[d][e];
        }
    }
    if (g == 0) {
        mine[0] = m;
        mine[1] = lsum[0];
    }
    __syncthreads();
    for (int i = tid; i < a.rows * D; i += 256) {
        const int r = i / D, d = i - r * D;
        const float* src = reinterpret_cast<const float*>(smem) + r * (D + 2);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = hv_max(top, src[w * 16 * (D + 2)]);
        const float ms = top == -INFINITY ? 0.f : top;
        float l = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* q = src + w * 16 * (D + 2);
            const float x = __builtin_amdgcn_exp2f((q[0] - ms) * a.c);
            l += x * q[1];
            o += x * q[2 + d];
        }
        if (a.splits > 1) {
            const long at = (((long)b * p.kv_heads + kvh) * a.rows + r) * a.splits + part.split;
            p.workspace[at * D + d] = o;
            if (d == 0) *reinterpret_cast<f32x2*>(hv_cross_weights(a) + at * 2) = f32x2{top, l};
        } else {
            int query, column;
            hv_cross_row(a, r, kvh, query, column);
            (p.O + (long)b * p.o_stride_b + (long)query * p.ldo + column)[d] = hv_f2bf(l == 0.f ? 0.f : o / l);
        }
    }
}

// joins the ranges of a row: o = sum_s o_s 2^((m_s - m) c) / sum_s l_s 2^((m_s - m) c); four values of a row per thread
template <int D>
__global__ __launch_bounds__(256) void hv_cross_attention_join_kernel(HvCrossArgs a) {
    const hv_cross_attention_params& p = a.p;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, item = i / (D / 4);
    const int d = (int)(i - item * (D / 4)) * 4;
    if (item >= (long)p.B * p.kv_heads * a.rows) return;
    const int r = (int)(item % a.rows);
    const int kvh = (int)(item / a.rows % p.kv_heads), b = (int)(item / a.rows / p.kv_heads);
    int len = p.kv_len ? p.kv_len[b] : p.Lk;
    len = len > p.Lk ? p.Lk : len;
    const int ranges = len <= a.per ? 1 : (len + a.per - 1) / a.per;  // those behind the entry's end wrote nothing
    const f32x2* const ml = reinterpret_cast<const f32x2*>(hv_cross_weights(a)) + item * a.splits;
    const float* const src = p.workspace + item * a.splits * D + d;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;  // ranges whose loads are in flight together
    for (int s0 = 0; s0 < ranges; s0 += U) {
        f32x2 w[U];
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u, ranges - 1);
            w[u] = ml[s];
            v[u] = *reinterpret_cast<const f32x4*>(src + (long)s * D);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) top = hv_max(top, w[u][0]);
        const float ms = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f((m - ms) * a.c);
        m = top;
        l *= old;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= old;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float x = s0 + u < ranges ? __builtin_amdgcn_exp2f((w[u][0] - ms) * a.c) : 0.f;
            l += x * w[u][1];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += x * v[u][e];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    int query, column;
    hv_cross_row(a, r, kvh, query, column);
    hv_st8(p.O + (long)b * p.o_stride_b + (long)query * p.ldo + column + d, u32x2{hv_pack2(o[0] * inv, o[1] * inv), hv_pack2(o[2] * inv, o[3] * inv)});
}

// sizes -> how the work is cut (also what hv_cross_attention_workspace answers from): -1 invalid, -2 head dim
static inline int hv_cross_attention_plan(const hv_cross_attention_params& p, HvCrossArgs& a) {
    if (p.B < 0 || p.Lq < 0 || p.Lk < 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads != 0) return -1;
    if (p.D != 40 && p.D != 64 && p.D != 80 && p.D != 128 && p.D != 160) return -2;
    const long rows = (long)p.Lq * (p.heads / p.kv_heads), pairs = (long)p.B * p.kv_heads;
    if (rows > 0x3fffffffL || pairs > 0x3fffffffL || p.Lk > 0x3fffffff) return -1;
    a.p = p;
    a.G = p.heads / p.kv_heads;
    a.rows = (int)rows;
    a.c = p.scale * 1.44269504088896341f;
    a.splits = a.run = a.per_wg = a.groups = 1;
    a.per = p.Lk;
    long units;
    if (p.Lk <= 96 && p.D <= 80 && p.heads % 4 == 0 && 4 % a.G == 0 && p.ldq < (1L << 24) && p.ldo < (1L << 24)) {
        // as many ranges of tiles as workgroups fit the chip at once: each pays for its states once
        a.kernel = 0;
        const int tile = HV_CROSS_FEW_ROWS(p.D);
        a.blocks = (p.Lq + tile - 1) / tile;
        const long lists = (long)p.B * (p.heads / 4), fit = 256L * (p.D == 40 ? 3 : 2);
        const long groups = lists > 0 && fit > lists ? fit / lists : 1;
        a.per_wg = (int)((a.blocks + groups - 1) / groups);
        if (a.per_wg < 1) a.per_wg = 1;
        a.groups = (a.blocks + a.per_wg - 1) / a.per_wg;
        units = lists * a.groups;
    } else {
        a.kernel = rows <= 16 ? 1 : rows <= 64 ? 2 : 3;
        const int block = a.kernel == 1 ? 16 : a.kernel == 2 ? 64 : 128, least = a.kernel == 1 ? 512 : 256;
        a.blocks = (int)((rows + block - 1) / block);
        const long base = pairs * a.blocks;
        if (base > 0 && base < 512 && p.Lk >= 2 * least) {
            // too few workgroups to fill the chip: cut the keys, to twice as many workgroups where entries may be of different lengths
            // (4 x 1536 queries, up to 4109 states, D = 80: ragged 71 us against 89, all full 102 against 94)
            const long want = ((p.kv_len ? 1024 : 512) + base - 1) / base, most = p.Lk / least;
            a.splits = (int)(want < most ? want : most);
            a.per = ((p.Lk + a.splits - 1) / a.splits + 127) / 128 * 128;
            a.splits = (p.Lk + a.per - 1) / a.per;
        }
        const long all = base * a.splits;
        a.run = (int)(all / 64 < 1 ? 1 : all / 64 < a.blocks ? all / 64 : a.blocks);  // at least 64 runs: 8 for each XCD
        units = all;
    }
    if (!hv_fits_launch(units + 8L * a.run, 256)) return -1;
    a.units = (int)units;
    return 0;
}

static inline long hv_cross_attention_floats(const HvCrossArgs& a) {
    return a.splits > 1 ? (long)a.p.B * a.p.kv_heads * a.rows * a.splits * (a.p.D + 2) : 0;
}

template <int D>
static inline void hv_cross_attention_launch_d(const HvCrossArgs& a, hipStream_t stream) {
    const int turn = 8 * a.run;
    const dim3 grid((unsigned)(((long)a.units + turn - 1) / turn * turn)), block(256);
    if constexpr (D <= 80) {
        if (a.kernel == 0) {
            const int nt = a.p.Lk <= 32 ? 2 : a.p.Lk <= 64 ? 4 : a.p.Lk <= 80 ? 5 : 6;
            hv_note("hv_cross_attention_few_kernel<%d,%d> | B=%d Lq=%d Lk=%d heads=%d/%d", D, nt, a.p.B, a.p.Lq, a.p.Lk, a.p.heads, a.p.kv_heads);
            if (nt == 2) hv_launch(hv_cross_attention_few_kernel<D, 2>, grid, block, stream, a);
            else if (nt == 4) hv_launch(hv_cross_attention_few_kernel<D, 4>, grid, block, stream, a);
            else if (nt == 5) hv_launch(hv_cross_attention_few_kernel<D, 5>, grid, block, stream, a);
            else hv_launch(hv_cross_attention_few_kernel<D, 6>, grid, block, stream, a);
            return;
        }
    }
    hv_note("hv_cross_attention_%s<%d> | B=%d Lq=%d Lk=%d heads=%d/%d ranges=%d", a.kernel == 1 ? "rows_kernel" : a.kernel == 2 ? "kernel<1>" : "kernel<2>",
            D, a.p.B, a.p.Lq, a.p.Lk, a.p.heads, a.p.kv_heads, a.splits);
    if (a.kernel == 1) hv_launch(hv_cross_attention_rows_kernel<D>, grid, block, stream, a);
    else if (a.kernel == 2) hv_launch(hv_cross_attention_kernel<D, 1>, grid, block, stream, a);
    else hv_launch(hv_cross_attention_kernel<D, 2>, grid, block, stream, a);
    if (a.splits > 1) {
        const long items = (long)a.p.B * a.p.kv_heads * a.rows;
        hv_note("hv_cross_attention_join_kernel<%d> | rows=%ld ranges=%d", D, items, a.splits);
        hv_launch(hv_cross_attention_join_kernel<D>, dim3((unsigned)((items * (D / 4) + 255) / 256)), block, stream, a);
    }
}

static inline long hv_cross_attention_workspace_of(const hv_cross_attention_params& p) {
    HvCrossArgs a;
    const int rc = hv_cross_attention_plan(p, a);
    return rc ? rc : hv_cross_attention_floats(a);
}

static inline int hv_cross_attention_launch(const hv_cross_attention_params& p, hipStream_t stream) {
    HvCrossArgs a;
    const int rc = hv_cross_attention_plan(p, a);
    if (rc) return rc;
    if (!(p.scale > 0.f) || p.scale > 1.0e30f) return -1;
    if (p.B == 0 || p.Lq == 0) return 0;
    const uint64_t addr = (uint64_t)p.Q | (uint64_t)p.K | (uint64_t)p.V | (uint64_t)p.O;
    const long strides = p.ldq | p.ldk | p.ldv | p.ldo | p.q_stride_b | p.k_stride_b | p.v_stride_b | p.o_stride_b;
    if ((addr & 15) != 0 || (strides & 7) != 0 || (strides | p.mask_stride_b) < 0) return -1;
    if (p.ldk > (1L << 24) || p.ldv > (1L << 24)) return -1;  // 64 rows within 32-bit offsets
    if (hv_cross_attention_floats(a) > p.workspace_floats || (a.splits > 1 && (p.workspace == nullptr || ((uint64_t)p.workspace & 15) != 0))) return -3;
    switch (p.D) {
        case 40: hv_cross_attention_launch_d<40>(a, stream); break;
        case 64: hv_cross_attention_launch_d<64>(a, stream); break;
        case 80: hv_cross_attention_launch_d<80>(a, stream); break;
        case 128: hv_cross_attention_launch_d<128>(a, stream); break;
        default: hv_cross_attention_launch_d<160>(a, stream); break;
    }
    return 0;
}
