// Block-quantised page chunks as f16 operand tiles of the tensor-core attention kernels.
#pragma once
#include "tc_common.cuh"

namespace b200kv {

__device__ inline void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- block-quantised chunk -> f16 operand tile(s) ----------------------------------------------------------------------
// Codes become exact f16 integers with byte permutes and one packed subtraction (0x6400 | u is the f16 1024 + u), the
// product with the f16 scale is one packed multiply, rounded once: RN_f16(code * scale), what rounding the reference's
// exact f32 product to f16 gives; for K a packed FMA returns the remainder code * scale - RN(code * scale), exact.
constexpr uint32_t H_MAGIC = 0x64646464u;  // source of the 0x64 high bytes
__device__ inline uint32_t hsub2(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&r;
}
__device__ inline uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*(const __half2*)&a, *(const __half2*)&b);
    return *(const uint32_t*)&r;
}
__device__ inline uint32_t hfma2_rem(uint32_t a, uint32_t b, uint32_t prod) {  // a * b - prod
    const __half2 r = __hfma2(*(const __half2*)&a, *(const __half2*)&b, __hneg2(*(const __half2*)&prod));
    return *(const uint32_t*)&r;
}
// where unit u (8 channels, 16 bytes) of row `row` lies in an operand tile
__device__ inline uint32_t tile_off(int u, int row) { return (u / 8) * (PAGE_TOKENS * 128) + row * 128 + (((u % 8) ^ (row & 7)) << 4); }

// Thread t of the FT converter threads takes item t % (D / 16) -- 16 channels, two units of 8 -- of every (16 FT / D)-th
// token: the 16 codes of an item come from one 16- or 8-byte load of a natural row (Q4_0: low and high nibbles of the same
// 8 bytes are the two units), or from 8 two-byte (Q8_1) / one-byte (Q4_0) loads of a permuted V row.  `lo_tile` (K): the
// tile that takes the remainders.  Rows from n_valid on are zero-filled.
template <int FMT, int D, int KV, int FT, bool FULL>
__device__ inline void convert_rows(const uint8_t* raw, uint8_t* hi_tile, uint8_t* lo_tile, int n_valid, int t) {
    constexpr bool PERM = v_permuted(FMT, D, KV), Q8 = FMT == B200KV_FMT_Q8_1, SPLIT = KV == 0;
    constexpr int ITEMS = D / 16, TLN = FT / ITEMS;
    constexpr uint32_t BIAS = Q8 ? 0x64806480u : 0x64086408u;  // f16 pair 1024 + 128 | 1024 + 8: what the codes are offset by
    const int item = t % ITEMS, tl = t / ITEMS;
    const __half* scales = (const __half*)(raw + PAGE_TOKENS * fmt_row_bytes(FMT, D));
    // The two units the item yields, and their blocks.  At head_dim 128 a quarter warp (one 16-byte store phase) is the eight
    // items of one token, four per 64-channel plane, and the planes lie a multiple of the bank width apart: if every item
    // stored its lower unit first, the planes would collide two ways in every store.  The items of the second plane
    // therefore take their units in the other order (`sw`): each phase then covers eight different 16-byte slots.
    const bool sw = D == 128 && (item & 4);
    int ua, ub;
    if (Q8 || PERM) ua = 2 * item + (sw ? 1 : 0), ub = 2 * item + (sw ? 0 : 1);
    else ua = 4 * (item / 2) + (item % 2) + (sw ? 2 : 0), ub = 4 * (item / 2) + (item % 2) + (sw ? 0 : 2);  // Q4_0 natural: bytes 16b + 8q .. hold channels 32b + 8q .. (low) and + 16 (high)
    const int blk_a = ua / 4, blk_b = ub / 4;
    const uint32_t sel_a = sw ? 0x4341u : 0x4240u, sel_b = sw ? 0x4240u : 0x4341u;  // permuted Q8_1 rows: which byte of a pair
    const int sh_a = sw ? 4 : 0, sh_b = sw ? 0 : 4;                                  // permuted Q4_0 rows: which nibble
#pragma unroll 4
    for (int tt = 0; tt < PAGE_TOKENS / TLN; tt++) {  // independent tokens: unrolled so that their loads and chains overlap
        const int tok = tt * TLN + tl;
        uint32_t ca[4], cb[4];  // f16 pairs: the codes of unit ua / ub as 1024 + u
        if constexpr (Q8 && !PERM) {
            const uint4 x = *(const uint4*)(raw + chunk_addr(FMT, D, KV, tok, 16 * item));
            const uint32_t w0 = sw ? x.z : x.x, w1 = sw ? x.w : x.y, w2 = sw ? x.x : x.z, w3 = sw ? x.y : x.w;
            ca[0] = __byte_perm(w0, H_MAGIC, 0x4140), ca[1] = __byte_perm(w0, H_MAGIC, 0x4342);
            ca[2] = __byte_perm(w1, H_MAGIC, 0x4140), ca[3] = __byte_perm(w1, H_MAGIC, 0x4342);
            cb[0] = __byte_perm(w2, H_MAGIC, 0x4140), cb[1] = __byte_perm(w2, H_MAGIC, 0x4342);
            cb[2] = __byte_perm(w3, H_MAGIC, 0x4140), cb[3] = __byte_perm(w3, H_MAGIC, 0x4342);
        } else if constexpr (Q8) {  // permuted V row: bytes 16r + 2 item, + 1 hold channels 16 item + r and + 8
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t h0 = *(const uint16_t*)(raw + chunk_addr(FMT, D, KV, tok, 16 * (2 * i) + 2 * item));
                const uint32_t h1 = *(const uint16_t*)(raw + chunk_addr(FMT, D, KV, tok, 16 * (2 * i + 1) + 2 * item));
                const uint32_t both = __byte_perm(h0, h1, 0x5410);  // [low r, high r, low r + 1, high r + 1]
                ca[i] = __byte_perm(both, H_MAGIC, sel_a), cb[i] = __byte_perm(both, H_MAGIC, sel_b);
            }
        } else if constexpr (!PERM) {  // Q4_0 natural row
            const uint2 x = *(const uint2*)(raw + chunk_addr(FMT, D, KV, tok, 16 * (item / 2) + 8 * (item % 2)));
            const uint32_t l0 = (x.x >> sh_a) & 0x0f0f0f0fu, h0 = (x.x >> sh_b) & 0x0f0f0f0fu, l1 = (x.y >> sh_a) & 0x0f0f0f0fu, h1 = (x.y >> sh_b) & 0x0f0f0f0fu;
            ca[0] = __byte_perm(l0, H_MAGIC, 0x4140), ca[1] = __byte_perm(l0, H_MAGIC, 0x4342);
            ca[2] = __byte_perm(l1, H_MAGIC, 0x4140), ca[3] = __byte_perm(l1, H_MAGIC, 0x4342);
            cb[0] = __byte_perm(h0, H_MAGIC, 0x4140), cb[1] = __byte_perm(h0, H_MAGIC, 0x4342);
            cb[2] = __byte_perm(h1, H_MAGIC, 0x4140), cb[3] = __byte_perm(h1, H_MAGIC, 0x4342);
        } else {  // Q4_0 permuted V row: byte 8r + item holds channel 16 item + r (low nibble) and + 8 (high nibble)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t b0 = raw[chunk_addr(FMT, D, KV, tok, 8 * (2 * i) + item)], b1 = raw[chunk_addr(FMT, D, KV, tok, 8 * (2 * i + 1) + item)];
                const uint32_t both = b0 | (b1 << 16);
                ca[i] = ((both >> sh_a) & 0x000f000fu) | 0x64006400u, cb[i] = ((both >> sh_b) & 0x000f000fu) | 0x64006400u;
            }
        }
        const uint32_t sa16 = __half_as_ushort(scales[scale_index(FMT, D, KV, tok, blk_a)]);
        const uint32_t sb16 = __half_as_ushort(scales[scale_index(FMT, D, KV, tok, blk_b)]);
        const uint32_t sa = sa16 | (sa16 << 16), sb = sb16 | (sb16 << 16);
        uint32_t ha[4], hb[4], la[4], lb[4];
        const bool ok = FULL || tok < n_valid;  // a full page (all but, at most, the last) runs without the sixteen selects
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t xa = hsub2(ca[i], BIAS), xb = hsub2(cb[i], BIAS);  // the codes themselves
            ha[i] = ok ? hmul2(xa, sa) : 0u, hb[i] = ok ? hmul2(xb, sb) : 0u;
            if (SPLIT) la[i] = ok ? hfma2_rem(xa, sa, ha[i]) : 0u, lb[i] = ok ? hfma2_rem(xb, sb, hb[i]) : 0u;
        }
        *(uint4*)(hi_tile + tile_off(ua, tok)) = make_uint4(ha[0], ha[1], ha[2], ha[3]);
        *(uint4*)(hi_tile + tile_off(ub, tok)) = make_uint4(hb[0], hb[1], hb[2], hb[3]);
        if (SPLIT) {
            *(uint4*)(lo_tile + tile_off(ua, tok)) = make_uint4(la[0], la[1], la[2], la[3]);
            *(uint4*)(lo_tile + tile_off(ub, tok)) = make_uint4(lb[0], lb[1], lb[2], lb[3]);
        }
    }
}

template <int FMT, int D, int KV, int FT>
__device__ inline void convert_chunk(const uint8_t* raw, uint8_t* hi_tile, uint8_t* lo_tile, int n_valid, int t) {
    if (n_valid >= PAGE_TOKENS) convert_rows<FMT, D, KV, FT, true>(raw, hi_tile, lo_tile, n_valid, t);
    else convert_rows<FMT, D, KV, FT, false>(raw, hi_tile, lo_tile, n_valid, t);
}

}  // namespace b200kv
