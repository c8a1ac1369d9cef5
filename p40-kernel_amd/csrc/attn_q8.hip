// attn_q8.hip -- attention over 8-bit pages (bonsai_p40_attn_paged and
// bonsai_p40_attn_shared with kv_type Q8): a row of a page is d n, n whole numbers of 8
// bits, d its scale.  The pass over the keys, its two shapes (rows, keys), the split
// and the join are those of attn_paged.hip; here is what the bytes change.
//
//   Scores.  q . k_j = d_j (q . n_j): the product runs on whole numbers, v_mfma_i32
// 32x32x32 with K's bytes as they lie in LDS.  A row of q becomes whole numbers, too, of
// 16 bits (16-bit queries) or 24 (fp32), its largest element at 127/128 of their range,
// as 2 or 3 digits of 8 bits with signs: a MFMA a digit, exact 32-bit sums, one
// conversion at the end.  A MFMA of these does twice a f16 one's work in its time, so that
// 2 digits cost what one f16 term does, 3 what 1.5 do, and no byte of K is unpacked.  An
// element of q is off by up to 2^-15 or 2^-23 of the row's largest.
//   Values.  O = sum_j p_j d_j n_j: the scale goes into the weight, w_j = p_j d_j, and
// V's bytes become f16, which holds them exactly: one XOR, two permutations (1024 + 128 +
// n as f16 bits) and two packed additions make 4 of them.  w is rounded to f16 once (16-bit
// output; error as in attn_paged.hip), or is two terms of f16 whose second has sums of its
// own (fp32).
//   f16's range is short for p_j d_j.  So the weights are relative to what follows a tile's largest
// score and the log2 of its largest d together, which leaves w at most 2^15, and a key
// whose p d is 2^-25 of its row's largest has all of f16's digits.  That says nothing of l, in which a
// key counts whatever its d: with 32 keys of d = 0 before 32 of d = 2^30 and equal scores, sums that shared that
// reference lost the first ones.  So l has a reference 2^m of its own, the scores', and O's is 2^(m + g): 2^g takes a
// tile's sum of weights over to l, and at the end O to m.
//   No value of V is NaN or infinite by itself, so a key that is not seen needs no
// zeroed row: its weight is 0 and its d counts as 0.
//   Keys (decode) is bound by the stream of the pages, half of 16-bit ones': 64 sequences of
// 16384, bf16, 5.64 TB/s; 1 of 131071 66 us (16-bit pages 109), 32 of up to 12000 103 to 104
// (154), where the batch's ragged parts leave CUs idle at the end (MI355X, heads of 256).
//   Rows (prompts) is bound by instructions: a tile of 32 keys on 128 rows takes 1.38 us (16-bit
// queries, heads of 256; 16-bit pages 1.15), 1024 clocks of it MFMA, and a wave's 270 VALU and 56
// LDS instructions hardly run beside them; fp32 2.1 (1.97).  777 tokens of 16000 keys: 500 us with
// each wave unpacking all of V for itself, 484 with each unpacking its own keys for all, 475 with
// the loads and that under the products (16-bit pages 362); fp32 rows 700.
#include "attn_device.h"
#include "gemv_device.h"
#include "host_state.h"
#include "launch_rules.h"

#include <type_traits>

using namespace mixer;

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// 8 keys x 16 bytes per 16 lanes, transposed: lane i gets column i
__device__ __forceinline__ v2u read_tr8(const uint8_t * at) {
    typedef int i2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i2 lds_i2;
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2 *)at));
}
// 4 keys x 16 f16
__device__ __forceinline__ v2u read_tr16(const uint8_t * at) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at));
}
// 8 signed bytes as f16
__device__ __forceinline__ v8h unpack(v2u x) {
    const v2h off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    v4u r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = x[i / 2] ^ 0x80808080u;         // 128 + n
        const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, i % 2 ? 0x04030402u : 0x04010400u);
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, h) + off);
    }
    return __builtin_bit_cast(v8h, r);
}
__device__ __forceinline__ v16f mfma(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <int D, bool KEYS, bool WIDE>
struct Shape {
    // (keys, heads of 256: two workgroups of 2 waves share a CU, so that one loads while the other begins or ends)
    static constexpr int NW = KEYS && D == 256 ? 2 : 4, BM = KEYS ? 32 : 32 * NW;
    static constexpr int RB = D, TILE = 32 * RB;           // bytes of a key, of a tile of 32 keys
    static constexpr int SC = (KEYS ? 2 : NW) * 256;       // of its scales: 256 for the keys of one DMA instruction
    static constexpr int R = 4;                            // rows: tiles of K, and of V, in LDS
    static constexpr int OROW = D + 4;                     // floats of a row in the join
    static constexpr int JOIN = NW * 32 * OROW * 4 + NW * 32 * 12;
    static constexpr int SLOTS = KEYS ? NW * 4 : 2 * R;    // keys: two buffers of K and V a wave
    // heads of 256: the registers hold the other digits of q, the lowest is in LDS (keys: the waves' is the same, and
    // all write it)
    static constexpr bool QL = D == 256 && (WIDE || !KEYS);
    static constexpr int QT = 32 * D;                      // bytes of a digit of 32 rows
    // rows: two tiles of V in f16
    static constexpr int MAIN = SLOTS * TILE, SCALED = MAIN + SLOTS * SC, WIDENED = SCALED + (QL ? (KEYS ? 1 : NW) * QT : 0);
    static constexpr int ALL = WIDENED + (KEYS ? 0 : 2 * 2 * TILE);
    static constexpr int LDS = KEYS && JOIN > ALL ? JOIN : ALL;
};

// IO: type of queries and output
template <class IO, int D, bool KEYS, bool SHARED>
__global__ void __launch_bounds__(KEYS && D == 256 ? 128 : 256) attn_q8_kernel(AttnArgs a) {
    constexpr bool WIDE = std::is_same<IO, F32>::value;
    typedef Shape<D, KEYS, WIDE> Z;
    constexpr int NT = WIDE ? 3 : 2;                       // digits of q
    constexpr int U = D / 16;                              // 16-byte units of a key
    constexpr int RPI = 64 / U;                            // keys per DMA instruction
    constexpr int QS = D / 32, DT = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Z::LDS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, half = lane >> 5;
    const AttnPlace at = attn_place<SHARED>(&a);
    const int kvh = at.kvh;
    // one sequence: the entries of a wave's first keys are asked for beside starts
    int early0 = -1, early1 = -1;
    const bool early = KEYS && !SHARED && a.n_seq == 1 && a.cap > 0 && a.n_pages > 0;
    if (early) {
        const int key = at.split * a.chunk + 32 * wave, top = (a.cap >> a.page_log2) - 1;
        early0 = sload(a.table, min(key >> a.page_log2, top));
        early1 = sload(a.table, min((key + 16) >> a.page_log2, top));
    }
    AttnWork w;
    if (!attn_work<Z::BM, SHARED>(a, at, w)) return;
    const Tile & tl = w.tl;
    const int kv = w.kv, before = w.before, nk = w.nk, k0 = w.k0, k1 = w.k1;
    const int lo = SHARED ? w.lo : 0;                      // keys before it are not seen
    const int rows = tl.count * a.group, row0 = tl.index * Z::BM, last = min(row0 + Z::BM, rows) - 1;

    // this lane's row
    const int wrow = row0 + (KEYS ? 0 : 32 * wave);
    const int r = wrow + n;
    const bool live = r < rows;
    const int tok = live ? r / a.group : 0, head = kvh * a.group + (live ? r - tok * a.group : 0);
    const int vis = live ? keys_seen<SHARED>(before, kv, tok) : 0;
    const int64_t grow = (int64_t)(tl.first + tok);
    // the fewest keys any live row of the wave sees, and any of the workgroup; 0 rows: nothing to do but stage
    const bool work = wrow < rows;
    const int least = work ? __builtin_amdgcn_readfirstlane(keys_seen<SHARED>(before, kv, wrow / a.group)) : 0;
    const int first_vis = __builtin_amdgcn_readfirstlane(keys_seen<SHARED>(before, kv, row0 / a.group));

    // Q^T, byte j of half h: d = 32 step + 16 h + j (a lane without a row: the tile's first), asked for here and
    // made into digits when the first tiles are on their way
    typedef typename IO::elem elem;
    typedef elem row16 __attribute__((ext_vector_type(16)));
    row16 qx[QS];
    {
        const elem * const qp = reinterpret_cast<const elem *>(a.q) + grow * a.q_tok + (int64_t)head * D + 16 * half;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            typedef elem row_part __attribute__((ext_vector_type(16 / sizeof(elem))));
#pragma unroll
            for (int i = 0; i < (int)sizeof(elem); ++i) {
                const row_part x = reinterpret_cast<const row_part *>(qp + 32 * s)[i];
#pragma unroll
                for (int j = 0; j < (int)(16 / sizeof(elem)); ++j) qx[s][i * (16 / sizeof(elem)) + j] = x[j];
            }
        }
    }
    v4i qf[NT][QS];
    uint8_t * const ql = lds + Z::SCALED + (KEYS ? 0 : wave * Z::QT) + 16 * lane;
    float c = a.c;
    // the factor of a row with a value that is not finite, which no other has: its sums mean nothing, and are NaN at the end
    // where it has seen a key
    constexpr float NOT_FINITE = 0x1p-149f;
    auto make_q = [&]() __attribute__((always_inline)) {
        // the largest magnitude's bits: they compare as the magnitudes do, and NaN is above infinity
        uint32_t big = 0;
        if constexpr (WIDE) {
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float f = qx[s][j];
                    const uint32_t x = __builtin_bit_cast(uint32_t, f) & 0x7fffffffu;
                    big = x > big ? x : big;
                }
        } else {
            typedef unsigned short u16 __attribute__((ext_vector_type(16)));
            typedef unsigned short u2 __attribute__((ext_vector_type(2)));
            u2 top = {0, 0};
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                const u16 x = __builtin_bit_cast(u16, qx[s]) & (unsigned short)0x7fff;
#pragma unroll
                for (int j = 0; j < 16; j += 2) top = __builtin_elementwise_max(top, (u2){x[j], x[j + 1]});
            }
            const unsigned short t = top[0] > top[1] ? top[0] : top[1];
            big = __builtin_bit_cast(uint32_t, IO::to(__builtin_bit_cast(elem, t)));
        }
        const uint32_t other = __shfl_xor(big, 32);
        big = other > big ? other : big;
        // times 2^k 127/128, so that the largest is 127/128 of 2^15 (2^23) at most: digits of -128 .. 127 hold it
        constexpr int TOP = NT == 3 ? 22 : 14;
        const int e = max((int)(big >> 23), TOP + 1);
        const float up = __builtin_bit_cast(float, (uint32_t)(254 + TOP - min(e, 254)) << 23) * (127.0f / 128.0f);
        // (the factor of a row next to 0 may come out as 0, which times a score of -inf is none)
        c = big >= 0x7f800000u ? NOT_FINITE : fmaxf(c * __builtin_bit_cast(float, (uint32_t)(min(e, 254) - TOP) << 23) * (128.0f / 127.0f), 0x1p-148f);
#pragma unroll
        for (int s = 0; s < QS; ++s)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // the whole number, its digits' bytes 128 up (of 16 bits: behind the point of 1.5 x 2^23, whose own
                    // low bits are 0)
                    const float f = IO::to(qx[s][j + i]);
                    if constexpr (NT == 3) v[i] = (uint32_t)(int)rintf(f * up) + 0x808080u;
                    else v[i] = __builtin_bit_cast(uint32_t, fmaf(f, up, 12582912.0f)) + 0x8080u;
                }
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    // byte k of each, without the 128
                    const uint32_t p = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u + 0x0101u * k);
                    const uint32_t q = __builtin_amdgcn_perm(v[3], v[2], 0x04000c0cu + 0x01010000u * k);
                    qf[k][s][j / 4] = (int)((p | q) ^ 0x80808080u);
                }
                if (Z::QL && j == 12) *reinterpret_cast<v4i *>(ql + 1024 * s) = qf[0][s];
            }
    };

    // ---- staging
    const int64_t trow = (int64_t)tl.seq * a.table_stride;
    auto swz_k = [](int key) { return (key / (16 / U)) & (U - 1); };
    auto swz_v = [](int key) {
        return U >= 16 ? 2 * (key & 3) | (key & 8) : U >= 8 ? (key & 2) | ((key >> 1) & 4) : (key >> 2) & 2;
    };
    // a page is one buffer: this head's rows are at head_at, their scales at scale_at
    auto swz_w = [](int key) { return U >= 16 ? (key & 7) * 4 : U >= 8 ? (key & 3) * 4 : ((key >> 1) & 1) * 4; };   // (units of 8 f16)
    const int in_page = (1 << a.page_log2) - 1, range = (int)a.scales + (a.n_kv << a.page_log2) * 4;
    const int head_at = kvh * (int)a.head_bytes, scale_at = (int)a.scales + (kvh << a.page_log2) * 4;
    auto page = [&](const uint8_t * base, int id) __attribute__((always_inline)) {
        return buffer_of(base + (int64_t)id * a.page_bytes, range);
    };
    // N keys of one page from `key` on to dst; place: that of the first among 16, as far as the swizzle (of K: swz, or
    // V's where the waves split the keys, or none) looks.  16 bytes a lane, or 4 where that is more than there are
    auto stage_n = [&](auto count, __amdgpu_buffer_rsrc_t from, int key, int place, uint8_t * dst, bool swz) __attribute__((always_inline)) {
        constexpr int N = decltype(count)::value, SIZE = N >= RPI ? 16 : 4, I = N * Z::RB / (64 * SIZE);
        const int first = head_at + (key & in_page) * Z::RB;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            // (the place of the lane's bytes in LDS, and theirs in the page, from a key that all lanes' begin at)
            const int at = SIZE * lane, kr = at / Z::RB, whole = i * 64 * SIZE / Z::RB, sw = place + whole + kr;
            const int off = kr * Z::RB + 16 * (at % Z::RB / 16 ^ (swz ? swz_k(sw) : KEYS ? swz_v(sw) : 0)) + at % 16;
            if constexpr (SIZE == 16) dma16(from, dst + i * 1024, off, first + whole * Z::RB);
            else dma4(from, dst + i * 256, off, first + whole * Z::RB);
        }
    };
    // Their scales, which a lane each brings.  The others ask for what is out of the buffer, for which nothing is read:
    // were they masked, the compiler may put the DMA instructions behind it into both sides of the branch
    auto stage_scales = [&](auto count, __amdgpu_buffer_rsrc_t from, int key, uint8_t * dst) __attribute__((always_inline)) {
        const int off = lane < decltype(count)::value ? 4 * lane : 0x7fffff00;
        dma4(from, dst, off, scale_at + 4 * (key & in_page));
    };

    // ---- one sub-tile of 32 keys
    const int l16 = lane & 15, vkey = 4 * half + ((l16 >> 1) & 3) + 8 * (l16 >> 3), vcol = (lane >> 4) & 1;
    uint32_t kat = n * Z::RB + 16 * (half ^ swz_k(n));
    uint32_t vat = vkey * Z::RB + 16 * (vcol ^ swz_v(vkey)) + 8 * (l16 & 1);
    auto k_frag = [&](const uint8_t * kb, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4i *>(kb + (kat ^ (32 * i)));
    };
    // keys 16 g + 4 half + j % 4 + 8 (j / 4) of d = 32 d + lane % 32
    auto v_frag = [&](const uint8_t * vb, int d, int g) __attribute__((always_inline)) {
        return read_tr8(vb + (vat ^ (32 * d)) + 16 * g * Z::RB);
    };
    // the scales of this lane's 16 keys
    auto scales4 = [&](const uint8_t * sb, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4f *>(sb + (KEYS ? 256 * (i / 2) + 32 * (i % 2) : 256 * i) + 16 * half);
    };
    auto scales = [&](const uint8_t * sb, v16f & x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4f y = scales4(sb, i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = y[j];
        }
    };
    // A sum of 256 products of digits is up to 2^22, 2^8 times that and another fit.  CHAIN: the highest digit's sums are
    // taken up 2^8 before the next digit's come into them, which saves the registers of one
    constexpr bool CHAIN = Z::QL && NT == 3;
    constexpr int NA = CHAIN ? 2 : NT;
    auto whole = [&](const v16i (&x)[NA], int i) __attribute__((always_inline)) {
        const float hi = (float)(CHAIN ? x[1][i] : (x[NA - 1][i] << 8) + x[NA - 2][i]);
        return NT == 3 ? fmaf(hi, 256.0f, (float)x[0][i]) : hi;
    };
    // step t of the product of a tile of K: fragment kf, lowest digit lf where LDS holds it
    constexpr int STEPS = CHAIN ? 2 * QS : QS;
    auto digits = [&](v16i (&x)[NA], v4i kf, v4i lf, int t) __attribute__((always_inline)) {
        if constexpr (CHAIN) {
            if (t < QS) {
                x[1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf, qf[2][t], x[1], 0, 0, 0);
                if (t == QS - 1) x[1] <<= 8;
            } else {
                x[0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf, lf, x[0], 0, 0, 0);
                x[1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf, qf[1][t - QS], x[1], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int k = NT - 1; k >= 0; --k)
                x[k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf, Z::QL && k == 0 ? lf : qf[k][t], x[k], 0, 0, 0);
        }
    };
    auto low_at = [](int t) { return CHAIN ? t - QS : t; };   // the step of the lowest digit, from 0 on
    // the scores of a tile, in whole numbers, at once
    auto product = [&](v16i (&x)[NA], const uint8_t * kb, const uint8_t * qlow) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NA; ++k) x[k] = v16i{};
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            digits(x, k_frag(kb, t % QS), Z::QL && low_at(t) >= 0 ? *reinterpret_cast<const v4i *>(qlow + 1024 * low_at(t)) : v4i{}, t);
        }
    };
    auto over_halves = [&](float mx) __attribute__((always_inline)) {
        const uint32_t x = __builtin_bit_cast(uint32_t, mx);
        const auto both = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        uint32_t p = both[0], q = both[1];
        asm("" : "+v"(p), "+v"(q));                        // they differ, though the operands do not
        return fmaxf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q));
    };
    // a row's largest score, in units of log2
    auto largest = [&](const v16f & s) __attribute__((always_inline)) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        return over_halves(mx) * c;
    };
    // log2 of the largest of the scales
    auto log_of = [&](float mx) __attribute__((always_inline)) {
        constexpr float least = 0x1p-100f;
        return __builtin_amdgcn_logf(fmaxf(over_halves(mx), least));
    };
    auto log_scale = [&](const v16f & vs) __attribute__((always_inline)) {
        float mx = fabsf(vs[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fabsf(vs[i]));
        return log_of(mx);
    };
    // what is not seen: scores -inf, scales 0; holes: bit g: the 16 keys from 16 g on are absent
    auto mask = [&](v16f & s, v16f & vs, int key0, int holes) __attribute__((always_inline)) {
        const int from = SHARED ? lo - key0 - 4 * half : 0, to = vis - key0 - 4 * half;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            // places from .. from + count are seen (SHARED), or 0 .. count
            const int count = holes >> g & 1 ? 0 : max(to - from, 0);
#pragma unroll
            for (int i = 8 * g; i < 8 * g + 8; ++i) {
                const uint32_t j = 8 * (i / 4) + i % 4 - from;
                s[i] = j >= (uint32_t)count ? -INFINITY : s[i];
                vs[i] = j >= (uint32_t)count ? 0.0f : vs[i];
            }
        }
    };
    // whether the row sees a key of the sub-tile
    auto sees = [&](int key0, int holes) __attribute__((always_inline)) {
        return (max(key0, lo) < (SHARED ? min(vis, key0 + 16) : vis) && !(holes & 1)) || (max(key0 + 16, lo) < vis && !(holes & 2));
    };
    v16f o[DT];
    auto clear = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);                 // (not before the queries are digits, as registers go)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            o[d] = v16f{};
            asm volatile("" : "+v"(o[d]));
        }
    };
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v16f{};
    // limit, ref, FAR and LEAST as in attn_paged.hip, where m follows the scores.  Here l is relative to 2^m, m the largest
    // score, whole, less a lag of up to LAG_L; O, and the weights that are made for it, to 2^(m + g), m + g following a tile's
    // largest score and the log2 of its largest d together, so that p d, which becomes f16, is up to 2^(UP + LAG), and 2^UP for
    // a key that has both (one of nearly all the weight is not rounded then).  g is in steps of 2^-16: m + g, and what these
    // change by, are exact where scores are below 128 (log2), and 2^g takes a tile's sum of weights over to l.  A d below 2^-100
    // counts as that: a weight is 2^115 at most, so that 16 of them add up, and with d up to 2^80 the smallest that fp32
    // holds is 2^-57 of its row's largest; l is below 2^40, O at its end below 2^127, for 2^31 keys
    constexpr float UP = 11.0f, LAG = 4.0f, LAG_L = 8.0f, LEAST = -3e38f, FAR = 1048576.0f, LOW_UP = 2048.0f;
    float m = -INFINITY, l = 0.0f, limit = -INFINITY, ref = 0.0f, g = 0.0f;
    // mx, lv: a tile's largest score, log2 of its largest d
    auto follow = [&](v16f & s, float mx, float lv) __attribute__((always_inline)) {
        if (__any(mx + lv > limit || mx - m > LAG_L)) {
            const float m2 = fmaxf(m, floorf(mx));
            const bool none = m2 == -INFINITY, near = fabsf(m2) < FAR;
            const float base = none ? 0.0f : m2, fall = none ? 0.0f : m - base;
            float g2 = fmaxf(g + fall, rintf((mx - base + lv) * 65536.0f) * (1.0f / 65536.0f) - UP);
            if (!near) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = s[i] * c;
                    asm("" : "+v"(x));                     // (no fma)
                    s[i] = (x - base) / c;
                }
            }
            ref = near ? m2 + g2 : g2;
            limit = near ? ref + (UP + LAG) : -INFINITY;
            if (near) g2 = ref - m2;                       // (as that was rounded)
            const float alpha = __builtin_amdgcn_exp2f(g + fall - g2);
            m = m2;
            g = g2;
            l *= __builtin_amdgcn_exp2f(fall);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
    };
    constexpr int NP = NT - 1;                             // f16 terms of a weight
    // weight e of a sub-tile into its operand; p goes to sum
    auto weight = [&](float s, float vs, v8h (&pf)[NP][2], int e, float & sum) __attribute__((always_inline)) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s, c, -ref));
        sum += p;
        float f = p * vs;
        if (NP == 2) asm("" : "+v"(f));                    // (both terms are of one f: not the product's f16 and then f's)
        const _Float16 x = (_Float16)f;
        pf[0][e / 8][e % 8] = x;
        if constexpr (NP == 2) pf[1][e / 8][e % 8] = (_Float16)((f - (float)x) * LOW_UP);
    };
    auto add_low = [&](const v16f & low, v16f & to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = fmaf(low[i], 1.0f / LOW_UP, to[i]);
    };

    if constexpr (!KEYS) {
        // As in attn_paged.hip: the scores of tile j + 1 beside the weights of tile j, K and V (and with K the scales
        // of both) in rings of R tiles.  V's bytes become f16 in LDS once for the four waves, each of which takes the
        // keys that it loaded itself, a tile ahead: where each wave unpacks all of a tile for itself it
        // has that many more VALU instructions, and these and the MFMAs of a wave hardly run side by side
        constexpr int R = Z::R, OWN = 32 / Z::NW, PER = 2 * (OWN >= RPI ? OWN / RPI : OWN * Z::RB / 256) + 2;   // keys, and DMA instructions, of a wave a tile
        const std::integral_constant<int, OWN> own_keys;
        const int own = wave * OWN, nt = (k1 - k0 + 31) / 32;
        uint8_t * const kring = lds, * const vring = lds + R * Z::TILE, * const ksring = lds + Z::MAIN, * const vsring = ksring + R * Z::SC;
        uint8_t * const wide_v = lds + Z::WIDENED;
        uint32_t hq = 0;                                   // holes, 2 bits a tile, the latest taken lowest
        int id = 0;                                        // the page of this wave's keys of the next tile
        const int second = own >= 16 ? -1 : 0;
        int raw0 = 0, raw1 = 0;
        const int top = max(nk - 1, 0) >> a.page_log2;
        const int32_t * const row = a.table + trow;
        auto ask = [&](int t) __attribute__((always_inline)) {
            const int key = k0 + 32 * t;
            raw0 = sload(row, min(key >> a.page_log2, top));
            raw1 = sload(row, min((key + 16) >> a.page_log2, top));
        };
        auto take = [&](int t) __attribute__((always_inline)) {
            const int key = k0 + 32 * t;
            const bool no0 = (key >= nk) | ((uint32_t)raw0 >= (uint32_t)a.n_pages);
            const bool no1 = (key + 16 >= nk) | ((uint32_t)raw1 >= (uint32_t)a.n_pages);
            hq = hq << 2 | (no0 ? 1 : 0) | (no1 ? 2 : 0);
            id = (no0 ? 0 : raw0 & ~second) + (no1 ? 0 : raw1 & second);   // (no page: any, of which nothing is seen)
        };
        // (this wave's place in a tile is computed anew each time: held for every slot it would take 24 registers)
        auto place = [&]() __attribute__((always_inline)) {
            int x = own;
            asm volatile("" : "+s"(x));
            return x;
        };
        auto stage_k = [&](int t, uint8_t * kt, uint8_t * ks) __attribute__((always_inline)) {
            const int at = place(), key = k0 + 32 * t + at;
            const auto from = page(a.k, id);
            stage_n(own_keys, from, key, own & 15, kt + at * Z::RB, true);
            stage_scales(own_keys, from, key, ks + at * (256 / OWN));
        };
        auto stage_v = [&](int t, uint8_t * vt, uint8_t * vs) __attribute__((always_inline)) {
            const int at = place(), key = k0 + 32 * t + at;
            const auto from = page(a.v, id);
            stage_n(own_keys, from, key, 0, vt + at * Z::RB, false);
            stage_scales(own_keys, from, key, vs + at * (256 / OWN));
        };
        // this wave's keys of a tile of V, a unit of 16 bytes a lane and step, to f16
        constexpr int UNITS = OWN * U, WS = UNITS < 64 ? 1 : UNITS / 64;
        const bool widens = UNITS >= 64 || lane < UNITS;
        // (fp32 rows of 256: the address of unit lane + 64, which is 4 keys on, where the swizzle differs in one bit, is made
        // from that of unit lane each time, as registers go: 777 tokens of 16000 keys up to 2 % faster than with two addresses.
        // 16-bit rows have the registers: 478 us, 487 with one)
        constexpr int WA = Z::QL && WIDE ? 1 : WS;
        static_assert(WA == WS || (WS == 2 && U == 16), "");
        uint32_t wat[WA];
#pragma unroll
        for (int i = 0; i < WA; ++i) {
            const int unit = lane + 64 * i, key = own + unit / U;
            wat[i] = key * 2 * Z::RB + 16 * ((2 * (unit % U)) ^ swz_w(key));
        }
        auto bytes_of = [&](const uint8_t * from, int i) __attribute__((always_inline)) {
            return *reinterpret_cast<const v4u *>(from + own * Z::RB + 1024 * i + 16 * lane);
        };
        // half h of unit i
        auto widen = [&](v4u x, uint8_t * to, int i, int h) __attribute__((always_inline)) {
            const v8h w = unpack((v2u){x[2 * h], x[2 * h + 1]});
            const uint32_t at = i < WA ? wat[i < WA ? i : 0] ^ (16 * h) : (wat[0] ^ (16 * h + 256)) + 8 * Z::RB;
            if (widens) *reinterpret_cast<v8h *>(to + at) = w;
        };
        // V in f16: keys 16 g + 4 half + j % 4 + 8 (j / 4) of d = 32 d + lane % 32
        const int wkey = 4 * half + (l16 >> 2), wcol = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
        const uint32_t fat = wkey * 2 * Z::RB + 16 * (wcol ^ swz_w(wkey)) + 8 * (l16 & 1);
        auto w_frag = [&](const uint8_t * vb, int d, int g) __attribute__((always_inline)) {
            const uint8_t * const at = vb + (fat ^ (64 * d)) + 16 * g * 2 * Z::RB;
            const v2u x = read_tr16(at), y = read_tr16(at + 8 * 2 * Z::RB);
            return __builtin_bit_cast(v8h, (v4u){x[0], x[1], y[0], y[1]});
        };
        v16f s, vs;                                        // the tile's scores, its scales of V
        float mx, lv;                                      // their largest, log2 of the largest
        // that the buffers differ has to be said, else every read of LDS waits for the DMA
        auto step = [&](auto edge, auto steady, uint8_t * __restrict__ kw, uint8_t * __restrict__ ksw, uint8_t * __restrict__ vw,
                        uint8_t * __restrict__ vsw, const uint8_t * __restrict__ kr, const uint8_t * __restrict__ ksr,
                        const uint8_t * __restrict__ v8r, const uint8_t * __restrict__ vsr, const uint8_t * __restrict__ vr,
                        uint8_t * __restrict__ v16w, const uint8_t * __restrict__ qlow, float bottom, int j) __attribute__((always_inline)) {
            constexpr bool EDGE = decltype(edge)::value;
            constexpr int KA = 2, VA = Z::QL && WIDE ? 2 : 4;   // fragments are read so many steps before they are used
            v4i kf[KA], lf[KA];
            auto k_read = [&](int i) __attribute__((always_inline)) {
                kf[i % KA] = k_frag(kr, i % QS);
                if (Z::QL && low_at(i) >= 0) lf[i % KA] = *reinterpret_cast<const v4i *>(qlow + 1024 * low_at(i));
            };
#pragma unroll
            for (int i = 0; i < KA; ++i) k_read(i);
            __builtin_amdgcn_sched_barrier(0);
            take(j + R);
            ask(j + R + 1);
            v4u bytes[WS];
            auto ask_bytes = [&]() __attribute__((always_inline)) {
                asm volatile("");                          // (on either side of the branch, not before it)
#pragma unroll
                for (int i = 0; i < WS; ++i) bytes[i] = bytes_of(v8r, i);
            };
            if (!work) {
                if (steady || j + R < nt) {
                    stage_k(j + R, kw, ksw);
                    stage_v(j + R, vw, vsw);
                }
                ask_bytes();
#pragma unroll
                for (int i = 0; i < 2 * WS; ++i) widen(bytes[i / 2], v16w, i / 2, i % 2);
                return;
            }
            // (three digits and two terms leave registers for one unit at a time)
            constexpr bool LATE = Z::QL && WIDE;
            if (!LATE) ask_bytes();
            const int key = k0 + 32 * j, holes = hq >> (2 * R) & 3;
            if (EDGE || holes) {
                mask(s, vs, key, holes);
                mx = largest(s);
                lv = log_scale(vs);
                if (sees(key, holes)) mx = fmaxf(mx, LEAST);
            }
            follow(s, mx, lv);
            constexpr int E = 16 / STEPS;
            float sum[2] = {0.0f, 0.0f};
            v8h vf[VA], pf[NP][2];
            v16i next[NA];
            v16f low;
            constexpr int KQ = Z::QL ? 2 : 4;              // scales of K in registers, 4 keys each
            v4f ks[KQ];
#pragma unroll
            for (int k = 0; k < NA; ++k) next[k] = v16i{};
            // a block's second term follows at once, where it has sums of its own
            auto v_read = [&](int i) __attribute__((always_inline)) {
                vf[i % VA] = NP == 2 ? w_frag(vr, i / 2, i % 2) : w_frag(vr, i % DT, i / DT);
            };
#pragma unroll
            for (int e = 0; e < E; ++e) weight(s[e], vs[e], pf, e, sum[e & 1]);
            __builtin_amdgcn_sched_barrier(0);
            // lgkmcnt(0): with a scalar load under way the waits below could not count
            __builtin_amdgcn_s_waitcnt(0xC07F);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                digits(next, kf[i % KA], lf[i % KA], i);
#pragma unroll
                for (int e = (i + 1) * E; e < (i + 2) * E && e < 16; ++e) weight(s[e], vs[e], pf, e, sum[e & 1]);
                if (i + KA < STEPS) k_read(i + KA);
                // (the last steps ask for the first fragments of V)
                constexpr int ASK = STEPS < VA ? STEPS : VA, EACH = VA / ASK;
                if (i >= STEPS - ASK) {
#pragma unroll
                    for (int x = 0; x < EACH; ++x) v_read((i - (STEPS - ASK)) * EACH + x);
                }
                // the loads of the tile R ahead, under the MFMAs
                if (i == 0 && (steady || j + R < nt)) stage_k(j + R, kw, ksw);
                if (i == STEPS / 2 && (steady || j + R < nt)) stage_v(j + R, vw, vsw);
                __builtin_amdgcn_sched_barrier(0);
            }
            l = fmaf(sum[0] + sum[1], __builtin_amdgcn_exp2f(g), l);
#pragma unroll
            for (int i = 0; i < KQ; ++i) ks[i] = scales4(ksr, i);
            scales(vsr, vs);
            // O takes them, and between the MFMAs the next scores are put together, their largest and that of the scales found
            float big[2] = {bottom, bottom}, lvs[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                const v8h vx = vf[i % VA];
                if constexpr (NP == 2) {
                    const int d = i / 2, g = i % 2;
                    if (g == 0) {
                        o[d] = mfma(vx, pf[0][g], o[d]);
                        if (d > 0) add_low(low, o[d - 1]);
                    }
                    low = mfma(vx, pf[1][g], g ? low : v16f{});
                    if (g == 1) o[d] = mfma(vx, pf[0][g], o[d]);
                } else {
                    o[i % DT] = mfma(vx, pf[0][i / DT], o[i % DT]);
                }
                if (i + VA < 2 * DT) v_read(i + VA);
                // V of the next tile becomes f16
                constexpr int EVERY = 2 * DT / (2 * WS);
                if (LATE && i % (2 * EVERY) == 0) bytes[0] = bytes_of(v8r, i / EVERY / 2);
                if (i % EVERY == (LATE ? EVERY / 2 : 0)) widen(bytes[LATE ? 0 : i / EVERY / 2], v16w, i / EVERY / 2, i / EVERY % 2);
#pragma unroll
                for (int e = i * 8 / DT; e < (i + 1) * 8 / DT; ++e) {
                    s[e] = whole(next, e) * ks[e / 4 % KQ][e % 4];
                    if (e % 4 == 3 && e / 4 + KQ < 4) ks[e / 4] = scales4(ksr, e / 4 + KQ);
                    big[e & 1] = fmaxf(big[e & 1], s[e]);
                    lvs[e & 1] = fmaxf(lvs[e & 1], fabsf(vs[e]));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (NP == 2) add_low(low, o[DT - 1]);
            mx = over_halves(fmaxf(big[0], big[1])) * c;
            lv = log_of(fmaxf(lvs[0], lvs[1]));
        };
        if (nt > 0) {
            ask(0);
#pragma unroll
            for (int t = 0; t < R; ++t) {
                take(t);
                ask(t + 1);
                if (t < nt) {
                    stage_k(t, kring + t * Z::TILE, ksring + t * Z::SC);
                    stage_v(t, vring + t * Z::TILE, vsring + t * Z::SC);
                }
            }
            make_q();
            clear();
            if (nt >= R) pq2::wait_vmcnt<(R - 1) * PER>();
            else pq2::wait_vmcnt<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < 2 * WS; ++i) widen(bytes_of(vring, i / 2), wide_v, i / 2, i % 2);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            {
                v16i x[NA];
                product(x, kring, ql);
                v16f ks;
                scales(ksring, ks);
                scales(vsring, vs);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = whole(x, i) * ks[i];
            }
            const float bottom = LEAST / fmaxf(c, 1.0f);   // (times c: finite)
            mx = fmaxf(largest(s), LEAST);
            lv = log_scale(vs);
            // tiles that every row sees whole, then those at the edge
            const int plain = SHARED && k0 < lo ? 0 : max(min(nt, (first_vis - k0) / 32), 0);
            // (steady: every load that a tile can start is there; R of them at a time, with the rings' places
            // known to the compiler)
            auto pass = [&](auto edge, auto steady, int slot, int j) __attribute__((always_inline)) {
                const int after = slot + 1 == R ? 0 : slot + 1;
                if (steady || j - 1 + R < nt) pq2::wait_vmcnt<(R - 2) * PER>();
                else pq2::wait_vmcnt<0>();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();              // the tiles are there, and all are done with the last ones
                asm volatile("" ::: "memory");
                step(edge, steady, kring + slot * Z::TILE, ksring + slot * Z::SC, vring + slot * Z::TILE, vsring + slot * Z::SC,
                     kring + after * Z::TILE, ksring + after * Z::SC, vring + after * Z::TILE, vsring + after * Z::SC,
                     wide_v + slot % 2 * 2 * Z::TILE, wide_v + (1 - slot % 2) * 2 * Z::TILE, ql, bottom, j);
            };
            int j = 0;
            const int all = min(plain, nt - R);
#pragma clang loop unroll(disable)
            for (; j + R <= all; j += R) {
                pass(std::false_type{}, std::true_type{}, 0, j);
                pass(std::false_type{}, std::true_type{}, 1, j + 1);
                pass(std::false_type{}, std::true_type{}, 2, j + 2);
                pass(std::false_type{}, std::true_type{}, 3, j + 3);
            }
            int slot = 0;
#pragma clang loop unroll(disable)
            for (; j < plain; ++j, slot = slot + 1 == R ? 0 : slot + 1) pass(std::false_type{}, std::false_type{}, slot, j);
#pragma clang loop unroll(disable)
            for (; j < nt; ++j, slot = slot + 1 == R ? 0 : slot + 1) pass(std::true_type{}, std::false_type{}, slot, j);
        }
    } else {
        uint8_t * const mine = lds + wave * 4 * Z::TILE, * const msc = lds + Z::MAIN + wave * 4 * Z::SC;
        auto page_of = [&](int key, bool have, int id) {
            if (key >= nk) return -1;
            if (!have) id = sload(a.table, trow + (key >> a.page_log2));
            return id >= 0 && id < a.n_pages ? id : -1;
        };
        // K of tile t + 2 is asked for when the scores of tile t are made, V when its sums are, so that one to two tiles
        // are under way (4 waves a workgroup: both asked for at the start of tile t + 1 measured the same, 32 sequences of
        // up to 12000 keys 105 us; two workgroups a CU of 2 waves 101)
        constexpr int HALF = 16 / RPI, NK = 2 * HALF + 4, NV = 2 * HALF;   // DMA instructions of a tile of K, of V
        const std::integral_constant<int, 16> half_tile;
        auto find = [&](int key, bool have, int (&to)[2]) __attribute__((always_inline)) {
            to[0] = page_of(key, have, early0);
            to[1] = page_of(key + 16, have, early1);
        };
        // (K brings the scales of both)
        auto stage_k = [&](int key, const int (&from)[2], uint8_t * to, uint8_t * sc) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const auto kp = page(a.k, max(from[g], 0));
                stage_n(half_tile, kp, key + 16 * g, 0, to + 16 * g * Z::RB, true);
                stage_scales(half_tile, kp, key + 16 * g, sc + 256 * g);
                stage_scales(half_tile, page(a.v, max(from[g], 0)), key + 16 * g, sc + Z::SC + 256 * g);
            }
        };
        auto stage_v = [&](int key, const int (&from)[2], uint8_t * to) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 2; ++g) stage_n(half_tile, page(a.v, max(from[g], 0)), key + 16 * g, 0, to + 16 * g * Z::RB, false);
        };
        constexpr int STRIDE = 32 * Z::NW;
        // kb, sc, vb: this tile's, which then take the one after the next's; ids: the pages of its halves, then of that one's
        auto step = [&](uint8_t * kb, uint8_t * sc, uint8_t * vb, int (&ids)[2], int key) __attribute__((always_inline)) {
            const bool next = key + STRIDE < k1, more = key + 2 * STRIDE < k1;
            // (fp32 rows of 256: the fragments' 16 addresses are made anew, as registers for them there are none)
            if (Z::QL) asm volatile("" : "+v"(kat), "+v"(vat));
            const int holes = (ids[0] < 0 ? 1 : 0) | (ids[1] < 0 ? 2 : 0);
            // behind K: V, and K and V of the next tile
            if (next) pq2::wait_vmcnt<NK + 2 * NV>();
            else pq2::wait_vmcnt<NV>();
            asm volatile("" ::: "memory");
            v16f s, vs;
            {
                v16i x[NA];
                v16f ks;
                auto get = [&]() __attribute__((always_inline)) {
                    scales(sc, ks);
                    scales(sc + Z::SC, vs);
                };
                if (!Z::QL) get();
                product(x, kb, ql);
                if (Z::QL) {
                    __builtin_amdgcn_sched_barrier(0);
                    get();
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = whole(x, i) * ks[i];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // its reads are done
            if (more) {
                find(key + 2 * STRIDE, false, ids);
                stage_k(key + 2 * STRIDE, ids, kb, sc);
            }
            float mx;
            if (key + 32 > least || holes || (SHARED && key < lo)) {
                mask(s, vs, key, holes);
                mx = largest(s);
                if (sees(key, holes)) mx = fmaxf(mx, LEAST);
            } else {
                mx = fmaxf(largest(s), LEAST);
            }
            follow(s, mx, log_scale(vs));
            v8h pf[NP][2];
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 16; ++e) weight(s[e], vs[e], pf, e, sum[e & 1]);
            l = fmaf(sum[0] + sum[1], __builtin_amdgcn_exp2f(g), l);
            asm volatile("" : "+v"(l));                    // (here, not behind the product, up to which 16 weights would be kept)
            // behind V: K and V of the next tile, K of the one after
            if (more) pq2::wait_vmcnt<2 * NK + NV>();
            else if (next) pq2::wait_vmcnt<NK + NV>();
            else pq2::wait_vmcnt<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const v8h v0 = unpack(v_frag(vb, d, 0)), v1 = unpack(v_frag(vb, d, 1));
                if constexpr (NP == 2) {
                    v16f low = mfma(v0, pf[1][0], v16f{});
                    low = mfma(v1, pf[1][1], low);
                    o[d] = mfma(v0, pf[0][0], o[d]);
                    o[d] = mfma(v1, pf[0][1], o[d]);
                    add_low(low, o[d]);
                } else {
                    o[d] = mfma(v0, pf[0][0], o[d]);
                    o[d] = mfma(v1, pf[0][1], o[d]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) stage_v(key + 2 * STRIDE, ids, vb);
        };
        int key = k0 + 32 * wave, ids[2] = {-1, -1}, next[2] = {-1, -1}, at = 0;
        if (key < k1) {
            find(key, early, ids);
            stage_k(key, ids, mine, msc);
            stage_v(key, ids, mine + Z::TILE);
        }
        if (key + STRIDE < k1) {
            find(key + STRIDE, false, next);
            stage_k(key + STRIDE, next, mine + 2 * Z::TILE, msc + 2 * Z::SC);
            stage_v(key + STRIDE, next, mine + 3 * Z::TILE);
        }
        make_q();
        clear();
#pragma clang loop unroll(disable)
        for (; key < k1; key += STRIDE, at ^= 1) {
            step(mine + at * 2 * Z::TILE, msc + at * 2 * Z::SC, mine + at * 2 * Z::TILE + Z::TILE, ids, key);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int x = ids[g];
                ids[g] = next[g];
                next[g] = x;
            }
        }
    }
    if (c == NOT_FINITE && m > -INFINITY) l = NAN;
    l += __shfl_xor(l, 32);
    const float gain = __builtin_amdgcn_exp2f(g);          // takes O over to 2^m (keys: where the waves are joined)
    if (!KEYS)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= gain;

    // (arguments that only this end of the kernel needs, read again rather than held all along)
    LateArgs * const z = late_args();
    const int part = attn_part<SHARED>(z, attn_place<SHARED>(z));

    const int n_part = SHARED ? z->n_split1 + z->n_split : z->n_split;
    const bool parts = SHARED || z->n_split > 1;
    const int64_t all_rows = (int64_t)z->n_tok * z->n_head;
    float * const pml = z->part + (int64_t)n_part * all_rows * D;
    if constexpr (!KEYS) {
        if (!live) return;
        const int64_t row = grow * z->n_head + head;
        const float f = parts ? 1.0f : over(m, l);
        float * const po = z->part + ((int64_t)part * all_rows + row) * D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = o[d][4 * q + j] * f;
                const int at = 32 * d + 8 * q + 4 * half;
                if (parts) store_row<F32>(po + at, x);
                else store_row<IO>(reinterpret_cast<elem *>(z->out) + grow * z->out_tok + (int64_t)head * D + at, x);
            }
        if (parts && half == 0)
            *reinterpret_cast<float2 *>(pml + 2 * ((int64_t)part * all_rows + row)) =
                make_float2(m, l);
    } else {
        // join the waves: [wave][row][D], [wave][row] (m, l) and [wave][row] 2^g
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        float * const jo = reinterpret_cast<float *>(lds);
        float2 * const ml = reinterpret_cast<float2 *>(lds + Z::NW * 32 * Z::OROW * 4);
        float * const gains = reinterpret_cast<float *>(ml + Z::NW * 32);
        if (live) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<v4f *>(jo + (wave * 32 + n) * Z::OROW + 32 * d + 8 * q + 4 * half) =
                        (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
            if (half == 0) {
                ml[wave * 32 + n] = make_float2(m, l);
                gains[wave * 32 + n] = gain;
            }
        }
        __syncthreads();
        constexpr int E = D / 64;
        for (int i = wave; i <= last - row0; i += Z::NW) {
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int k = 0; k < Z::NW; ++k) mm = fmaxf(mm, ml[k * 32 + i].x);
            const float to = mm == -INFINITY ? 0.0f : mm;
            float x[E] = {};
#pragma unroll
            for (int k = 0; k < Z::NW; ++k) {
                const float2 e = ml[k * 32 + i];
                const float wt = __builtin_amdgcn_exp2f(e.x - to), wo = wt * gains[k * 32 + i];
                ll = fmaf(e.y, wt, ll);
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] = fmaf(jo[(k * 32 + i) * Z::OROW + lane * E + j], wo, x[j]);
            }
            const int rr = row0 + i, t = rr / z->group, h = kvh * z->group + rr - t * z->group;
            const int64_t g = tl.first + t, row = g * z->n_head + h;
            if (parts) {
                store_row<F32>(z->part + ((int64_t)part * all_rows + row) * D + lane * E, x);
                if (lane == 0) *reinterpret_cast<float2 *>(pml + 2 * ((int64_t)part * all_rows + row)) = make_float2(mm, ll);
            } else {
                const float inv = over(mm, ll);
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] *= inv;
                store_row<IO>(reinterpret_cast<elem *>(z->out) + g * z->out_tok + (int64_t)h * D + lane * E, x);
            }
        }
    }
}

template <class IO, int D, bool KEYS, bool SHARED>
int launch(AttnArgs & a, bool first, bool own, hipStream_t s) {
    AttnArgs b = a;
    b.blocks1 = first ? (unsigned)((int64_t)a.tiles1 * a.n_split1 * a.n_kv) : 0;
    const int64_t blocks = b.blocks1 + (own ? (int64_t)a.tiles * a.n_split * a.n_kv : 0);
    hipLaunchKernelGGL((attn_q8_kernel<IO, D, KEYS, SHARED>), dim3((unsigned)blocks), dim3(64 * Shape<D, KEYS, false>::NW), 0, s, b);
    return (int)hipGetLastError();
}
template <class IO, int D, bool SHARED>
int launch_k(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    int e = 0;
    const bool both = SHARED && l.keys1 == l.keys &&
                      pq2::attn_one_launch((int64_t)a.tiles1 * a.n_split1 * a.n_kv, (int64_t)a.tiles * a.n_split * a.n_kv);
    if (SHARED && !both)
        e = l.keys1 ? launch<IO, D, true, SHARED>(a, true, false, s) : launch<IO, D, false, SHARED>(a, true, false, s);
    if (e) return e;
    e = l.keys ? launch<IO, D, true, SHARED>(a, both, true, s) : launch<IO, D, false, SHARED>(a, both, true, s);
    return e || !l.parts ? e : launch_join<IO, D, SHARED>(a, l.keys ? Shape<D, true, false>::BM : Shape<D, false, false>::BM, s);
}
template <class IO, int D>
int launch_s(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    return l.shared ? launch_k<IO, D, true>(l, a, s) : launch_k<IO, D, false>(l, a, s);
}
template <class IO>
int launch_d(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    return l.head_dim == 256 ? launch_s<IO, 256>(l, a, s) : l.head_dim == 128 ? launch_s<IO, 128>(l, a, s) : launch_s<IO, 64>(l, a, s);
}

}  // namespace

int mixer::attn_q8_launch(AttnArgs & a, const AttnLaunch & l, hipStream_t s) {
    return l.io_type == BONSAI_P40_F32 ? launch_d<F32>(l, a, s) : l.io_type == BONSAI_P40_F16 ? launch_d<F16>(l, a, s)
                                                                                             : launch_d<BF16>(l, a, s);
}
