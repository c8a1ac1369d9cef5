// attn_paged.hip -- attention of every sequence's new tokens over its pages
// (bonsai_p40_attn_paged): one token (decode), a few, or a prompt chunk, ragged,
// grouped heads, causal.
//
//   o_t = sum_{j < p_t} softmax(scale q_t . k_j) v_j,   p_t = kv_len - n_new + t + 1
//
// One pass over the keys with the running maximum m and sum l of the softmax
// (in units of log2, so that exp2 takes them):
//   m' = max(m, c s),  p = 2^(c s - m'),  l' = l 2^(m - m') + sum p,  O' = O 2^(m - m') + p V.
//
// A row of the products is a (token, query head) pair: the heads that share a
// key/value head share its tiles, so a decode step of 6 heads is 6 rows and a
// chunk of n tokens 6 n.  Both products run transposed on v_mfma 32x32x16:
//   S^T (32 keys x 32 rows) = K . Q^T,   O^T (32 d x 32 rows) += V^T . P^T.
// A lane then holds 16 keys of ONE row, so that maximum, sum and rescaling are a
// lane's own (one exchange with lane ^ 32), and the P it computes is the operand
// of the second product as it stands: element j of half h is key 4 h + j % 4 +
// 8 (j / 4) there, an order of the contraction that V^T is read in too
// (ds_read_b64_tr_b16 transposes 4 keys x 16 d on the way out of LDS).
// K and V tiles reach LDS by DMA, 16-byte units XOR-swizzled by the key on the
// source side so that neither read meets a bank twice.
//
// Two shapes of workgroup, both on tiles of 32 keys:
//   rows: a wave per 32 rows (64 or 128 a workgroup), all on the same tiles, which
//     come through rings of 3 or 4 in LDS: prompts, bound by the matrix cores;
//   keys: 32 rows, each wave its own tiles, double-buffered, joined in LDS at the
//     end: decode, bound by the stream of K and V.
// Either splits the keys over workgroups where there are too few rows to fill the
// card; attn_join_kernel adds the parts.
//   SHARED: batches that share a prefix (attn_device.h).  A workgroup has rows of a whole group
// and its shared keys, or a sequence's and its own, which need not begin with a tile: what is
// before them is masked.  64 sequences behind 16000 keys, up to 500 each, bf16, 24 heads of 256:
// 43 us for the prefix, 23 for the own keys, 10 to join (MI355X); attn_paged over the same tables reads the prefix 64 times.
//
// fp32 queries and output (the activations' type) keep fp32 accuracy: Q and P
// are split into 2 f16 terms (22 bits) or 3 bf16 terms (24 bits) and the products
// summed in fp32.  16-bit ones round P once to the pages' type, as its relative
// error is that of the output's own rounding (norm of the error over that of the result,
// scores of one size: bf16 1.7e-3 by the output alone, 2.3e-3 with P's; f16 2.1e-4, 2.9e-4).
//   f16's smallest step is 2^-24, and a row may have one key of nearly all the weight
// before thousands that share the rest.  So with f16 pages m is kept 11 below, and P
// is 2^11 at the maximum, up to 2^15 as m follows with a lag of up to 4 (bf16, which
// has fp32's range: 0 and 8; l, O and the parts scale alike): one term is 11 bits of
// weights down to 2^-25 of the row's largest, below that off by up to 2^-36 of it.
// The second term, up to 2^-12 of its weight, is taken 2^11 up, in sums of its own
// for a tile that O gets 2^-11 of: 22 bits down to 2^-25, 2^-47 below.  In the first
// one's sums it would have that one's steps: with a key e^12 above 4000 others, of
// value 0, the result would be off by 1.2e-6 (6e-8 so), e^18 by 3.2e-4 (2e-7).  It
// costs 128 FMA a tile of heads of 256: fp32 queries, f16 pages, 2048 tokens 117 -> 129
// us (MI355X), 777 of 16000 keys 560 -> 617, 9 ragged sequences with heads of 128 183 ->
// 208.  One term, lags of 2, 4 and 8 (13, 11 and 7 below), 2048 tokens: 79.7, 77.6 and 77.4 us.
#include "gemv_device.h"
#include "host_state.h"
#include "launch_rules.h"
#include "attn_device.h"

#include <type_traits>

using namespace mixer;

namespace {

template <class T>
__device__ __forceinline__ v16f mfma(typename T::frag a, typename T::frag b, v16f c);
template <>
__device__ __forceinline__ v16f mfma<F16>(v8h a, v8h b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ v16f mfma<BF16>(v8b a, v8b b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 4 keys x 16 d per 16 lanes, transposed: lane i gets column i
__device__ __forceinline__ v2u read_tr(const uint8_t * at) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at));
}

template <class T, int D, int NT, bool KEYS>
struct Shape {
    // waves: with heads of 256, LDS has two buffers of 32 keys for 2 waves, or 64 rows of two terms of Q
    static constexpr int NW = D == 256 && (KEYS || NT == 3) ? 2 : 4;
    static constexpr int BM = KEYS ? 32 : 32 * NW;
    // fp32 queries of 256: the registers hold one term of Q, the others are in LDS
    static constexpr bool QL = NT > 1 && D == 256;
    static constexpr int QR = QL ? 1 : NT;                 // terms in registers
    static constexpr int RB = 2 * D;                       // bytes of a key
    static constexpr int TILE = 32 * RB;                   // of a tile of 32 keys
    static constexpr int R = QL ? 3 : 4;                   // rows: tiles of K, and of V, in LDS
    static constexpr int OROW = D + 4;                     // floats of a row in the join
    static constexpr int JOIN = NW * 32 * OROW * 4 + NW * 32 * 8;
    static constexpr int MAIN = KEYS ? NW * 4 * TILE : 2 * R * TILE;   // keys: two buffers of K and V a wave
    static constexpr int QT = 2 * 32 * D;                  // bytes of a term of 32 rows
    static constexpr int ALL = MAIN + (NT - QR) * (KEYS ? QT : NW * QT);
    static constexpr int LDS = KEYS && JOIN > ALL ? JOIN : ALL;
};

template <class T, int D, int NT, bool KEYS, bool SHARED>
__global__ void __launch_bounds__(D == 256 && (KEYS || NT == 3) ? 128 : 256) attn_kernel(AttnArgs a) {
    typedef Shape<T, D, NT, KEYS> Z;
    typedef typename T::elem elem;
    typedef typename T::frag frag;
    constexpr int U = D / 8;                               // 16-byte units of a key
    constexpr int RPI = 64 / U;                            // keys per DMA instruction
    constexpr int QS = D / 16, DT = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Z::LDS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, half = lane >> 5;
    const AttnPlace at = attn_place<SHARED>(&a);
    const int kvh = at.kvh;
    // one sequence: its row of the table is known (and there is one, where there are pages), and the entries of a wave's first keys are asked for beside starts
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
    // the fewest keys any live row of the wave sees; 0 rows: nothing to do but stage
    const bool work = wrow < rows;
    const int least = work ? __builtin_amdgcn_readfirstlane(keys_seen<SHARED>(before, kv, wrow / a.group)) : 0;

    // the keys that all rows of the workgroup see
    const int first_vis = __builtin_amdgcn_readfirstlane(keys_seen<SHARED>(before, kv, row0 / a.group));

    // Q^T, element j of half h: d = 16 step + 8 h + j (a lane without a row: the tile's first).  fp32 queries
    // are asked for here, and made into terms when the first tiles are on their way
    typedef typename std::conditional<NT == 1, frag, v8f>::type raw;
    typedef typename std::conditional<NT == 1, elem, float>::type qelem;
    raw qx[QS];
    {
        const qelem * const qp = reinterpret_cast<const qelem *>(a.q) + grow * a.q_tok + (int64_t)head * D + 8 * half;
#pragma unroll
        for (int s = 0; s < QS; ++s) qx[s] = *reinterpret_cast<const raw *>(qp + 16 * s);
    }
    frag qf[Z::QR][QS];
    uint8_t * const ql = lds + Z::MAIN + (KEYS ? 0 : wave * (NT - Z::QR) * Z::QT) + 16 * lane;
    float c = a.c;
    constexpr bool LOW = NT == 2;                          // P's second term has sums of its own
    constexpr float UP = std::is_same<T, F16>::value ? 11.0f : 0.0f, LAG = UP > 0.0f ? 4.0f : 8.0f;
    constexpr float LOW_UP = 2048.0f;
    auto make_q = [&]() __attribute__((always_inline)) {
        if constexpr (NT == 1) {
#pragma unroll
            for (int s = 0; s < QS; ++s) qf[0][s] = qx[s];
        } else {
            float up = 1.0f;
            if constexpr (NT == 2) {
                // the row's largest element to 2^14 .. 2^15: f16 then holds 22 bits in two terms of elements down to
                // 2^-18 of it, and is off by up to 2^-40 of it below
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < QS; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(qx[s][j]));
                big = fmaxf(big, __shfl_xor(big, 32));
                const int e = (int)((__builtin_bit_cast(uint32_t, big) >> 23) & 255);
                if (e > 14 && e < 255) {
                    up = __builtin_bit_cast(float, (uint32_t)(268 - e) << 23);
                    c = fmaxf(c * __builtin_bit_cast(float, (uint32_t)(e - 14) << 23), 0x1p-149f);   // (0 times -inf is none)
                }
            }
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                frag low[NT];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float f = qx[s][j] * up;
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        const elem e = T::from(f);
                        if (k < Z::QR) qf[k][s][j] = e;
                        else low[k][j] = e;
                        f -= T::to(e);
                    }
                }
#pragma unroll
                for (int k = Z::QR; k < NT; ++k)
                    if (!KEYS || wave == 0) *reinterpret_cast<frag *>(ql + (k - Z::QR) * Z::QT + 1024 * s) = low[k];
            }
            if constexpr (Z::QL && KEYS) {                 // (rows: each wave reads its own)
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
        }
    };

    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v16f{};
    float m = -INFINITY, l = 0.0f;

    // ---- staging: 16 keys of K and V a call, all of one page
    const int64_t trow = (int64_t)tl.seq * a.table_stride;
    const int drow = lane / U, dunit = lane % U;
    auto swz_k = [](int key) { return U >= 16 ? key & 15 : (key >> 1) & 7; };
    auto swz_v = [](int key) { return U >= 32 ? (key & 7) * 4 : U >= 16 ? (key & 3) * 4 : ((key >> 1) & 1) * 4; };
    // the page of the 16 keys from `key` on; -1: none of them is to be read
    auto page_of = [&](int key, bool have, int id) {
        if (key >= nk) return -1;
        if (!have) id = sload(a.table, trow + (key >> a.page_log2));
        return id >= 0 && id < a.n_pages ? id : -1;
    };
    // N keys of one page from `key` on to dst; place: that of the first among 16, as far as the swizzle looks.
    // The page's rows of this head, and no others, are in range
    const uint8_t * const khead = a.k + (int64_t)kvh * a.head_bytes, * const vhead = a.v + (int64_t)kvh * a.head_bytes;
    const int in_page = (1 << a.page_log2) - 1, range = Z::RB << a.page_log2;
    auto stage_n = [&](auto count, const uint8_t * head, int id, int key, int place, uint8_t * dst, bool is_v) __attribute__((always_inline)) {
        const auto from = buffer_of(head + (int64_t)max(id, 0) * a.page_bytes, range);
        const int first = (key & in_page) * Z::RB;
        constexpr int N = decltype(count)::value / RPI;
        auto lane_off = [&](int i) __attribute__((always_inline)) {
            const int kr = place + i * RPI + drow;
            return drow * Z::RB + 16 * (dunit ^ (is_v ? swz_v(kr) : swz_k(kr)));
        };
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            dma16_at<0>(from, dst + i * 1024, lane_off(i), first + i * 1024);
            if constexpr (N > 1) dma16_at<1024>(from, dst + i * 1024, lane_off(i + 1), first + i * 1024);
            if constexpr (N > 2) {
                dma16_at<2 * 1024>(from, dst + i * 1024, lane_off(i + 2), first + i * 1024);
                dma16_at<3 * 1024>(from, dst + i * 1024, lane_off(i + 3), first + i * 1024);
            }
        }
    };
    // zero the rows [from, to) of V: p is 0 there, and 0 times what memory holds may be NaN
    auto zero_keys = [&](uint8_t * dst, int from, int to) {
        for (int i = from * U + lane; i < to * U; i += 64) *reinterpret_cast<v4u *>(dst + 16 * i) = v4u{};
    };

    // ---- one sub-tile of 32 keys: kb, vb its first keys in LDS, key0 its place
    // in the sequence, holes: bit g: the 16 keys from 16 g on are absent
    // the swizzle leaves the address of step i, or of the 32 d of block i, at one address XOR a constant
    const int l16 = lane & 15, vkey = 4 * half + (l16 >> 2), vcol = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    const uint32_t kat = n * Z::RB + 16 * (half ^ swz_k(n));
    // (V's place, VOFF behind K's, goes into its address: it is more than an instruction's offset holds)
    constexpr int VOFF = KEYS ? Z::TILE : Z::R * Z::TILE;
    uint32_t vat = VOFF + vkey * Z::RB + 16 * (vcol ^ swz_v(vkey)) + 8 * (l16 & 1);
    asm("" : "+v"(vat));
    auto k_frag = [&](const uint8_t * kb, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const frag *>(kb + (kat ^ (32 * i)));
    };
    // keys 16 g + 4 half + j % 4 + 8 (j / 4) of d = 32 d + lane % 32; kb: as for K
    auto v_frag = [&](const uint8_t * kb, int d, int g) __attribute__((always_inline)) {
        const uint8_t * const at = kb + (vat ^ (64 * d)) + 16 * g * Z::RB;
        const v2u x = read_tr(at), y = read_tr(at + 8 * Z::RB);
        return __builtin_bit_cast(frag, (v4u){x[0], x[1], y[0], y[1]});
    };
    auto scores = [&](const uint8_t * kb, const uint8_t * ql) __attribute__((always_inline)) {
        v16f s = {};
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            const frag kf = k_frag(kb, i);
#pragma unroll
            for (int k = NT - 1; k >= Z::QR; --k)
                s = mfma<T>(kf, *reinterpret_cast<const frag *>(ql + (k - Z::QR) * Z::QT + 1024 * i), s);
#pragma unroll
            for (int k = Z::QR - 1; k >= 0; --k) s = mfma<T>(kf, qf[k][i], s);
        }
        return s;
    };
    // scores that are not seen to -inf
    auto mask = [&](v16f & s, int key0, int holes) __attribute__((always_inline)) {
        if constexpr (SHARED) {
            int from = lo - key0 - 4 * half, to = vis - key0 - 4 * half;
            asm("" : "+v"(from));                          // (its part that all lanes share is not worth 16 scalars)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const uint32_t count = holes >> g & 1 ? 0 : max(to - from, 0);   // places from .. from + count are seen
#pragma unroll
                for (int i = 8 * g; i < 8 * g + 8; ++i)
                    if ((uint32_t)(8 * (i / 4) + i % 4 - from) >= count) s[i] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = 8 * (i / 4) + 4 * half + i % 4;
                if (key0 + j >= vis || (holes >> (j >> 4) & 1)) s[i] = -INFINITY;
            }
        }
    };
    // a row's largest score, in units of log2: half the keys are in lane ^ 32
    auto over_halves = [&](float mx) __attribute__((always_inline)) {
        const uint32_t x = __builtin_bit_cast(uint32_t, mx);
        const auto both = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        uint32_t lo = both[0], hi = both[1];
        asm("" : "+v"(lo), "+v"(hi));                      // they differ, though the operands do not
        return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)) * c;
    };
    auto largest = [&](const v16f & s) __attribute__((always_inline)) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        return over_halves(mx);
    };
    // whether the row sees a key of the sub-tile
    auto sees = [&](int key0, int holes) __attribute__((always_inline)) {
        return (max(key0, lo) < (SHARED ? min(vis, key0 + 16) : vis) && !(holes & 1)) || (max(key0 + 16, lo) < vis && !(holes & 2));
    };
    // m follows UP below the running maximum with a lag, so that the sums are rescaled seldom: at a largest score above
    // limit.  It is -inf while the row has seen no key, and finite behind that, whatever the scores (LEAST): l = 0 is then
    // 0 / 0.  ref: what the weights subtract.
    //   m is a product that was rounded, and one fma of a score less it is off by up to half its step: FAR from 0 that
    // is p far from 1, or past f16's end.  There each tile's scores are rounded like m first, as those of a softmax of
    // fp32 scores are, ref is 0, and P 1 at the maximum
    constexpr float LEAST = -3e38f, FAR = 1048576.0f;
    float limit = -INFINITY, ref = 0.0f;
    auto follow = [&](v16f & s, float mx) __attribute__((always_inline)) {
        if (__any(mx > limit)) {
            const bool near = fabsf(fmaxf(m, mx)) < FAR;
            const float m2 = fmaxf(m, near ? mx - UP : mx), base = m2 == -INFINITY ? 0.0f : m2;
            if (!near) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = s[i] * c;
                    asm("" : "+v"(x));                     // (no fma)
                    s[i] = (x - base) / c;
                }
            }
            limit = near ? m2 + (UP + LAG) : -INFINITY;
            ref = near ? m2 : 0.0f;
            const float alpha = __builtin_amdgcn_exp2f(m - base);
            m = m2;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
    };
    auto weights = [&](v16f & s) __attribute__((always_inline)) {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -ref));
            sum[i & 1] += s[i];
        }
        l += sum[0] + sum[1];
    };
    // where some rows of the wave see a key and others do not, p = 0 does not keep an infinity or NaN of V out
    // of the others' sums: bit k: key k of the sub-tile has one
    auto wild = [&](const uint8_t * vb) __attribute__((always_inline)) {
        typedef unsigned short u2 __attribute__((ext_vector_type(2)));
        constexpr uint32_t EXP = T::EXP * 0x10001u;
        u2 top = {0, 0};
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
            const v4u x = *reinterpret_cast<const v4u *>(vb + n * Z::RB + 16 * (half * (U / 2) + (i + n) % (U / 2)));
#pragma unroll
            for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u2, x[j] & EXP));
        }
        const uint64_t hit = __ballot(top[0] == T::EXP || top[1] == T::EXP);
        return (uint32_t)(hit | hit >> 32);
    };
    // those keys one by one, for the rows that see them; then their rows of V are zeroed.  mixed is uniform
    // over the waves that share the tile, and so is what is found
    auto apart = [&](const v16f & p, uint8_t * vb, int key0) __attribute__((always_inline)) {
        const uint32_t bad = wild(vb);
        if (!bad) return;
        for (uint32_t left = bad; left; left &= left - 1) {
            const int k = __builtin_ctz(left), at = (k & 3) + 4 * (k >> 3);
            float x = p[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) x = at == i ? p[i] : x;
            x = __shfl(x, n + 32 * (k >> 2 & 1));
            if (key0 + k < vis) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float v[4];
                        load_row<T>(reinterpret_cast<const elem *>(vb + k * Z::RB + 16 * ((4 * d + g) ^ swz_v(k)) + 8 * half), v);
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[d][4 * g + j] = fmaf(x, v[j], o[d][4 * g + j]);
                    }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (!KEYS) __builtin_amdgcn_s_barrier();           // all waves have what they need of these rows
        asm volatile("" ::: "memory");
        for (uint32_t left = bad; left; left &= left - 1)
            for (int i = lane; i < U; i += 64)
                *reinterpret_cast<v4u *>(vb + __builtin_ctz(left) * Z::RB + 16 * i) = v4u{};
    };
    // elements from .. to of a block of O get those of P's second term
    auto add_low = [&](const v16f & low, v16f & to, int first, int end) __attribute__((always_inline)) {
#pragma unroll
        for (int i = first; i < end; ++i) to[i] = fmaf(low[i], 1.0f / LOW_UP, to[i]);
    };
    auto values = [&](const v16f & p, const uint8_t * kb) __attribute__((always_inline)) {
        frag pf[NT][2];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float f = p[8 * g + j];
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    const elem e = T::from(f);
                    pf[k][g][j] = e;
                    f = LOW ? (f - T::to(e)) * LOW_UP : f - T::to(e);
                }
            }
        if constexpr (LOW) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const frag v0 = v_frag(kb, d, 0), v1 = v_frag(kb, d, 1);
                v16f low = mfma<T>(v0, pf[1][0], v16f{});
                low = mfma<T>(v1, pf[1][1], low);
                o[d] = mfma<T>(v0, pf[0][0], o[d]);
                o[d] = mfma<T>(v1, pf[0][1], o[d]);
                add_low(low, o[d], 0, 16);
            }
        } else {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const frag vf = v_frag(kb, d, g);
#pragma unroll
                    for (int k = NT - 1; k >= 0; --k) o[d] = mfma<T>(vf, pf[k][g], o[d]);
                }
        }
    };

    if constexpr (!KEYS) {
        // A tile of 32 keys at a time: while the matrix cores work on the scores of tile j + 1, the weights of
        // tile j are made, then O takes them.  R tiles of K and R of V are in LDS, the others on their way
        constexpr int R = Z::R, OWN = 32 / Z::NW, PER = 2 * OWN / RPI;   // keys, and DMA instructions, of a wave a tile
        const int own = wave * OWN, nt = (k1 - k0 + 31) / 32;
        uint8_t * const kring = lds, * const vring = lds + R * Z::TILE;
        uint32_t hq = 0;                                   // holes, 2 bits a tile, the latest taken lowest
        int idk = -1, idv = -1;                            // pages of this wave's keys of the next tiles of K and of V
        // the table's entries for tile t are asked for one tile before they are taken
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
            const bool ok0 = key < nk && (uint32_t)raw0 < (uint32_t)a.n_pages;
            const bool ok1 = key + 16 < nk && (uint32_t)raw1 < (uint32_t)a.n_pages;
            hq = hq << 2 | (ok0 ? 0 : 1) | (ok1 ? 0 : 2);
            idv = idk;
            idk = own < 16 ? (ok0 ? raw0 : -1) : (ok1 ? raw1 : -1);
        };
        auto stage = [&](const uint8_t * base, int id, int t, uint8_t * to, bool is_v) __attribute__((always_inline)) {
            int at = own;                                  // (SHARED: anew each time, as held for every slot it takes too many registers)
            if (SHARED) asm volatile("" : "+s"(at));
            stage_n(std::integral_constant<int, OWN>{}, base, id, k0 + 32 * t + at, at & 15, to + at * Z::RB, is_v);
        };
        // that the buffers differ has to be said, else every read of LDS waits for the DMA
        auto step = [&](auto edge, auto steady, uint8_t * __restrict__ kw, uint8_t * __restrict__ vw, const uint8_t * __restrict__ kr,
                        uint8_t * __restrict__ vr, const uint8_t * __restrict__ qlow, float bottom, v16f & s, float & mx, int j) __attribute__((always_inline)) {
            constexpr bool EDGE = decltype(edge)::value;
            // fragments are read AHEAD steps before they are used
            constexpr int AHEAD = Z::QL ? 2 : 4;
            frag kf[AHEAD], lf[AHEAD][NT];
            auto k_read = [&](int i) __attribute__((always_inline)) {
                kf[i % AHEAD] = k_frag(kr, i);
#pragma unroll
                for (int k = Z::QR; k < NT; ++k)
                    lf[i % AHEAD][k - Z::QR] = *reinterpret_cast<const frag *>(qlow + (k - Z::QR) * Z::QT + 1024 * i);
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) k_read(i);
            __builtin_amdgcn_sched_barrier(0);
            take(j + R);
            ask(j + R + 1);
            if (steady || j + R < nt) stage(khead, idk, j + R, kw, false);
            if (steady || j + R - 1 < nt) stage(vhead, idv, j + R - 1, vw, true);
            const int key = k0 + 32 * j, holes = hq >> (2 * R) & 3;
            const bool mixed = EDGE && key + 32 > first_vis && nk > max(first_vis, key);
            if (!work && !mixed) return;
            if (EDGE || holes) {
                mask(s, key, holes);
                mx = largest(s);
                if (sees(key, holes)) mx = fmaxf(mx, LEAST);
            }
            follow(s, mx);
            // the scores of the next tile, and between their MFMAs the weights of this one (E of a step)
            constexpr int E = 16 / QS > 0 ? 16 / QS : 1;
            float sum[2] = {0.0f, 0.0f};
            frag vf[AHEAD], pf[NT][2];
            // (heads of 256: one wave a SIMD, and room for two blocks' sums of the second term; else a block's go to O before the next)
            constexpr int LB = D == 256 ? 2 : 1;
            v16f next = {}, low[LB];
            // the blocks of V in the order of their products: a block's second term follows at once, where it has sums of its own
            auto v_read = [&](int i) __attribute__((always_inline)) {
                vf[i % AHEAD] = LOW ? v_frag(vr, i / 2, i % 2) : v_frag(vr, i % DT, i / DT);
            };
            // lgkmcnt(0): with a scalar load under way the waits below could not count
            __builtin_amdgcn_s_waitcnt(0xC07F);
#pragma unroll
            for (int i = 0; i < QS; ++i) {
#pragma unroll
                for (int k = NT - 1; k >= Z::QR; --k) next = mfma<T>(kf[i % AHEAD], lf[i % AHEAD][k - Z::QR], next);
#pragma unroll
                for (int k = Z::QR - 1; k >= 0; --k) next = mfma<T>(kf[i % AHEAD], qf[k][i], next);
                if (i + AHEAD < QS) k_read(i + AHEAD);
                else if (!EDGE) v_read(i + AHEAD - QS);
#pragma unroll
                for (int e = i * E; e < (i + 1) * E; ++e) {
                    s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, -ref));
                    sum[e & 1] += s[e];
                    float f = s[e];
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        const elem x = T::from(f);
                        pf[k][e / 8][e % 8] = x;
                        f = LOW ? (f - T::to(x)) * LOW_UP : f - T::to(x);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            l += sum[0] + sum[1];
            if (EDGE) {
                if (mixed) apart(s, vr + VOFF, key);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) v_read(i);
            }
            // O takes them, and between the MFMAs the largest of the next scores are found
            float top[2] = {bottom, bottom};
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                if constexpr (LOW) {
                    const int d = i / 2, g = i % 2;
                    if (LB == 1 && g == 0) {
                        o[d] = mfma<T>(vf[i % AHEAD], pf[0][g], o[d]);
                        if (d > 0) add_low(low[0], o[d - 1], 0, 16);
                    }
                    low[d % LB] = mfma<T>(vf[i % AHEAD], pf[1][g], g ? low[d % LB] : v16f{});
                    if (LB == 2 || g == 1) o[d] = mfma<T>(vf[i % AHEAD], pf[0][g], o[d]);
                    if (LB == 2 && d > 0) add_low(low[(d - 1) % LB], o[d - 1], 8 * g, 8 * g + 8);
                } else {
#pragma unroll
                    for (int k = NT - 1; k >= 0; --k) o[i % DT] = mfma<T>(vf[i % AHEAD], pf[k][i / DT], o[i % DT]);
                }
                if (i + AHEAD < 2 * DT) v_read(i + AHEAD);
#pragma unroll
                for (int e = i * 8 / DT; e < (i + 1) * 8 / DT; ++e) top[e & 1] = fmaxf(top[e & 1], next[e]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (LOW) add_low(low[(DT - 1) % LB], o[DT - 1], 0, 16);
            mx = over_halves(fmaxf(top[0], top[1]));
            s = next;
        };
        if (nt > 0) {
            ask(0);
#pragma unroll
            for (int t = 0; t < R; ++t) {
                take(t);
                ask(t + 1);
                if (t < nt) stage(khead, idk, t, kring + t * Z::TILE, false);
                if (t > 0 && t - 1 < nt) stage(vhead, idv, t - 1, vring + (t - 1) * Z::TILE, true);
            }
            make_q();
            if (nt >= R) pq2::wait_vmcnt<(R - 1) * PER>();
            else pq2::wait_vmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            v16f s = scores(kring, ql);
            const float bottom = LEAST / fmaxf(c, 1.0f);   // (times c: finite)
            float mx = fmaxf(largest(s), LEAST);
            // tiles that every row sees whole, then those at the edge
            const int plain = SHARED && k0 < lo ? 0 : max(min(nt, (first_vis - k0) / 32), 0);
            // (steady: every load that a tile can start is there; R of them at a time, with the rings' places
            // known to the compiler)
            auto pass = [&](auto edge, auto steady, int slot, int j) __attribute__((always_inline)) {
                const int after = slot + 1 == R ? 0 : slot + 1, before = slot == 0 ? R - 1 : slot - 1;
                if (steady || j - 1 + R < nt) pq2::wait_vmcnt<(R - 2) * PER>();
                else pq2::wait_vmcnt<0>();
                const int holes = hq >> (2 * R - 2) & 3, key = k0 + 32 * j + own;
                const bool hole = holes >> (own >> 4) & 1;
                if (SHARED && !steady && key < lo) zero_keys(vring + slot * Z::TILE + own * Z::RB, 0, min(lo - key, OWN));
                if (hole || (!steady && key + OWN > nk))
                    zero_keys(vring + slot * Z::TILE + own * Z::RB, hole ? 0 : iclamp(nk - key, 0, OWN), OWN);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();              // the tiles are there, and all are done with the last ones
                asm volatile("" ::: "memory");
                step(edge, steady, kring + slot * Z::TILE, vring + before * Z::TILE, kring + after * Z::TILE, lds + slot * Z::TILE,
                     ql, bottom, s, mx, j);
            };
            int j = 0;
            const int whole = min(plain, nt - R);
#pragma clang loop unroll(disable)
            for (; j + R <= whole; j += R) {
                pass(std::false_type{}, std::true_type{}, 0, j);
                pass(std::false_type{}, std::true_type{}, 1, j + 1);
                pass(std::false_type{}, std::true_type{}, 2, j + 2);
                if constexpr (R == 4) pass(std::false_type{}, std::true_type{}, 3, j + 3);
            }
            int slot = 0;
#pragma clang loop unroll(disable)
            for (; j < plain; ++j, slot = slot + 1 == R ? 0 : slot + 1) pass(std::false_type{}, std::false_type{}, slot, j);
#pragma clang loop unroll(disable)
            for (; j < nt; ++j, slot = slot + 1 == R ? 0 : slot + 1) pass(std::true_type{}, std::false_type{}, slot, j);
        }
    } else {
        uint8_t * const mine = lds + wave * 4 * Z::TILE;
        int id0 = -1, id1 = -1;
        auto stage = [&](int key, bool have, uint8_t * to) __attribute__((always_inline)) {
            id0 = page_of(key, have, early0);
            id1 = page_of(key + 16, have, early1);
            const std::integral_constant<int, 16> half_tile;
            stage_n(half_tile, khead, id0, key, 0, to, false);
            stage_n(half_tile, khead, id1, key + 16, 0, to + 16 * Z::RB, false);
            stage_n(half_tile, vhead, id0, key, 0, to + Z::TILE, true);
            stage_n(half_tile, vhead, id1, key + 16, 0, to + Z::TILE + 16 * Z::RB, true);
        };
        auto step = [&](uint8_t * __restrict__ next, uint8_t * __restrict__ cur, const uint8_t * __restrict__ qlow,
                        int key, int holes) __attribute__((always_inline)) {
            if (key + 32 * Z::NW < k1) stage(key + 32 * Z::NW, false, next);
            v16f s = scores(cur, qlow);
            float mx;
            if (key + 32 > least || holes || (SHARED && key < lo)) {
                mask(s, key, holes);
                mx = largest(s);
                if (sees(key, holes)) mx = fmaxf(mx, LEAST);
            } else {
                mx = fmaxf(largest(s), LEAST);
            }
            follow(s, mx);
            weights(s);
            if (key + 32 > first_vis && nk > max(first_vis, key)) apart(s, cur + Z::TILE, key);
            values(s, cur);
        };
        int key = k0 + 32 * wave, b = 0;
        if (key < k1) stage(key, early, mine);
        make_q();
#pragma clang loop unroll(disable)
        for (; key < k1; key += 32 * Z::NW, b ^= 1) {
            const int holes = (id0 < 0 ? 1 : 0) | (id1 < 0 ? 2 : 0);
            uint8_t * const cur = mine + b * 2 * Z::TILE;
            pq2::wait_vmcnt<0>();
            if (SHARED && key < lo) zero_keys(cur + Z::TILE, 0, min(lo - key, 32));
            if (holes || key + 32 > nk) {
                zero_keys(cur + Z::TILE, holes & 1 ? 0 : iclamp(nk - key, 0, 16), 16);
                zero_keys(cur + Z::TILE, holes & 2 ? 16 : iclamp(nk - key, 16, 32), 32);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // also: the other buffer's reads are done
            step(mine + (b ^ 1) * 2 * Z::TILE, cur, ql, key, holes);
        }
    }
    l += __shfl_xor(l, 32);

    // (SHARED: the arguments of this end of the kernel are read again rather than held all along)
    const auto z = args_of<SHARED>(a);
    const int part = attn_part<SHARED>(z, SHARED ? attn_place<SHARED>(z) : at);
    const int n_part = SHARED ? z->n_split1 + z->n_split : z->n_split;
    const bool parts = SHARED || z->n_split > 1;
    const int64_t all_rows = (int64_t)z->n_tok * z->n_head;
    if constexpr (!KEYS) {
        if (!live) return;
        const int64_t row = grow * z->n_head + head;
        const float inv = parts ? 1.0f : over(m, l);
        float * const po = z->part + ((int64_t)part * all_rows + row) * D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = o[d][4 * g + j] * inv;
                const int at = 32 * d + 8 * g + 4 * half;
                if (parts) store_row<F32>(po + at, x);
                else if constexpr (NT == 1)
                    store_row<T>(reinterpret_cast<elem *>(z->out) + grow * z->out_tok + (int64_t)head * D + at, x);
                else store_row<F32>(reinterpret_cast<float *>(z->out) + grow * z->out_tok + (int64_t)head * D + at, x);
            }
        if (parts && half == 0)
            *reinterpret_cast<float2 *>(z->part + (int64_t)n_part * all_rows * D + 2 * ((int64_t)part * all_rows + row)) =
                make_float2(m, l);
    } else {
        // join the waves: [wave][row][D] and [wave][row] (m, l)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        float * const jo = reinterpret_cast<float *>(lds);
        float2 * const ml = reinterpret_cast<float2 *>(lds + Z::NW * 32 * Z::OROW * 4);
        if (live) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<v4f *>(jo + (wave * 32 + n) * Z::OROW + 32 * d + 8 * g + 4 * half) =
                        (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
            if (half == 0) ml[wave * 32 + n] = make_float2(m, l);
        }
        __syncthreads();
        constexpr int E = D / 64;
        for (int i = wave; i <= last - row0; i += Z::NW) {
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int k = 0; k < Z::NW; ++k) mm = fmaxf(mm, ml[k * 32 + i].x);
            const float ref = mm == -INFINITY ? 0.0f : mm;
            float x[E] = {};
#pragma unroll
            for (int k = 0; k < Z::NW; ++k) {
                const float2 e = ml[k * 32 + i];
                const float w = __builtin_amdgcn_exp2f(e.x - ref);
                ll = fmaf(e.y, w, ll);
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] = fmaf(jo[(k * 32 + i) * Z::OROW + lane * E + j], w, x[j]);
            }
            const int rr = row0 + i, t = rr / z->group, h = kvh * z->group + rr - t * z->group;
            const int64_t g = tl.first + t, row = g * z->n_head + h;
            if (parts) {
                store_row<F32>(z->part + ((int64_t)part * all_rows + row) * D + lane * E, x);
                if (lane == 0)
                    *reinterpret_cast<float2 *>(z->part + (int64_t)n_part * all_rows * D +
                                                2 * ((int64_t)part * all_rows + row)) = make_float2(mm, ll);
            } else {
                const float inv = over(mm, ll);
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] *= inv;
                if constexpr (NT == 1)
                    store_row<T>(reinterpret_cast<elem *>(z->out) + g * z->out_tok + (int64_t)h * D + lane * E, x);
                else store_row<F32>(reinterpret_cast<float *>(z->out) + g * z->out_tok + (int64_t)h * D + lane * E, x);
            }
        }
    }
}

// Shared prefixes: their phase and that of the own keys in one launch where both have this shape, then the join
template <class T, int D, int NT, bool KEYS, bool SHARED>
int launch(AttnArgs & a, bool first, bool own, hipStream_t s) {
    typedef Shape<T, D, NT, KEYS> Z;
    AttnArgs b = a;
    b.blocks1 = first ? (unsigned)((int64_t)a.tiles1 * a.n_split1 * a.n_kv) : 0;
    const int64_t blocks = b.blocks1 + (own ? (int64_t)a.tiles * a.n_split * a.n_kv : 0);
    hipLaunchKernelGGL((attn_kernel<T, D, NT, KEYS, SHARED>), dim3((unsigned)blocks), dim3(64 * Z::NW), 0, s, b);
    return (int)hipGetLastError();
}
template <class T, int D, int NT, bool SHARED>
int launch_k(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    int e = 0;
    const bool both = SHARED && l.keys1 == l.keys &&
                      pq2::attn_one_launch((int64_t)a.tiles1 * a.n_split1 * a.n_kv, (int64_t)a.tiles * a.n_split * a.n_kv);
    if (SHARED && !both)
        e = l.keys1 ? launch<T, D, NT, true, SHARED>(a, true, false, s) : launch<T, D, NT, false, SHARED>(a, true, false, s);
    if (e) return e;
    e = l.keys ? launch<T, D, NT, true, SHARED>(a, both, true, s) : launch<T, D, NT, false, SHARED>(a, both, true, s);
    if (e || !l.parts) return e;
    typedef typename std::conditional<NT == 1, T, F32>::type TO;
    return launch_join<TO, D, SHARED>(a, l.keys ? Shape<T, D, NT, true>::BM : Shape<T, D, NT, false>::BM, s);
}
template <class T, int D, int NT>
int launch_s(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    return l.shared ? launch_k<T, D, NT, true>(l, a, s) : launch_k<T, D, NT, false>(l, a, s);
}
template <class T, int NT>
int launch_d(const AttnLaunch & l, AttnArgs & a, hipStream_t s) {
    return l.head_dim == 256 ? launch_s<T, 256, NT>(l, a, s) : l.head_dim == 128 ? launch_s<T, 128, NT>(l, a, s)
                                                                                 : launch_s<T, 64, NT>(l, a, s);
}

// 1: invalid, 0: nothing to do, -1: to be run
int check(const bonsai_p40_attn_paged_args * p) {
    if (!p) return 1;
    const int d = p->head_dim;
    if (d != 64 && d != 128 && d != 256) return 1;
    if (p->n_kv_head < 1 || p->n_head < 1 || p->n_head > 65536 || p->n_head % p->n_kv_head != 0) return 1;
    if (p->kv_type == BONSAI_P40_Q8 ? !is_type(p->io_type)
                                    : !is_half(p->kv_type) || (p->io_type != BONSAI_P40_F32 && p->io_type != p->kv_type))
        return 1;
    if (!is_pow2(p->page_size) || p->page_size < 16 || p->page_size > 65536) return 1;
    if (p->n_pages < 0 || p->n_pages > 0x7fffffff) return 1;
    if (!page_stride_ok(p->kv_type, p->page_stride, p->n_kv_head, p->page_size, d)) return 1;
    // (an 8-bit page is one buffer)
    if (p->kv_type == BONSAI_P40_Q8 && (int64_t)p->n_kv_head * p->page_size * (d + 4) > 0x7fffffff) return 1;
    const int per16 = 16 / type_bytes(p->io_type);
    if (p->q_tok < (int64_t)p->n_head * d || p->q_tok % per16 != 0) return 1;
    if (p->out_tok < (int64_t)p->n_head * d || p->out_tok % per16 != 0) return 1;
    if (!(p->scale > 0.0f) || !(p->scale < INFINITY)) return 1;
    if (p->max_pages < 0 || p->table_stride < p->max_pages || p->max_kv < 0) return 1;
    if (p->max_pages * (int64_t)p->page_size > 0x7fff0000) return 1;
    if (p->n_tok <= 0 || p->n_seq <= 0) return 0;
    if (p->n_tok > 0x7fffffff / p->n_head || p->n_seq > 0xffffff) return 1;
    if ((p->n_tok + p->n_seq) * (int64_t)p->n_head >= 1 << 24) return 1;    // a grid has fewer than 2^32 threads
    return -1;
}
// ... of the pointers
bool pointers_ok(const bonsai_p40_attn_paged_args * p) {
    if (pq2host::any_null(p->q, p->out, p->starts, p->kv_len)) return false;
    if (p->max_pages > 0 && p->n_pages > 0 && pq2host::any_null(p->k_pages, p->v_pages, p->table)) return false;
    return aligned(p->q, 16) && aligned(p->out, 16) && aligned(p->k_pages, 16) && aligned(p->v_pages, 16) &&
           aligned(p->workspace, 16) && aligned(p->table, 4) && aligned(p->starts, 4) && aligned(p->kv_len, 4);
}

struct Plan {
    bool keys;
    int tiles, chunk, n_split;
};
enum Keys { ALL, SHARED_KEYS, OWN_KEYS };
// n_seq sequences, or groups, of up to `most` keys
Plan plan_of(const bonsai_p40_attn_paged_args * p, int n_seq, int64_t most, Keys which = ALL) {
    const int group = p->n_head / p->n_kv_head;
    const int rows = p->head_dim == 256 && p->kv_type == BONSAI_P40_BF16 && p->io_type == BONSAI_P40_F32 ? 64 : 128;
    const int cus = pq2host::device_info().cus;
    const bool bytes = p->kv_type == BONSAI_P40_Q8;
    const pq2::AttnPlan a = which == OWN_KEYS
        ? pq2::attn_own_plan(p->n_tok, n_seq, group, p->n_kv_head, p->head_dim, most, rows, cus, bytes)
        : pq2::attn_plan(p->n_tok, n_seq, group, p->n_kv_head, p->head_dim, most, rows, cus, bytes, which == SHARED_KEYS);
    return {a.keys, (int)a.tiles, (int)a.chunk, (int)a.n_split};
}
int64_t most_keys(const bonsai_p40_attn_paged_args * p) {
    const int64_t cap = (int64_t)p->max_pages * p->page_size;
    return p->max_kv > 0 && p->max_kv < cap ? p->max_kv : cap;
}
int64_t part_bytes(const bonsai_p40_attn_paged_args * p, int n_part) {
    return n_part <= 1 ? 0 : (int64_t)n_part * p->n_tok * p->n_head * (p->head_dim + 2) * 4;
}

void fill(AttnArgs & a, const bonsai_p40_attn_paged_args * p, const Plan & pl) {
    const int el = p->kv_type == BONSAI_P40_Q8 ? 1 : 2;
    a = AttnArgs{};
    a.q = p->q;
    a.out = p->out;
    a.k = reinterpret_cast<const uint8_t *>(p->k_pages);
    a.v = reinterpret_cast<const uint8_t *>(p->v_pages);
    a.table = p->table;
    a.starts = p->starts;
    a.kv_len = p->kv_len;
    a.part = reinterpret_cast<float *>(p->workspace);
    a.q_tok = p->q_tok;
    a.out_tok = p->out_tok;
    a.page_bytes = p->page_stride * el;
    a.head_bytes = (int64_t)p->page_size * p->head_dim * el;
    a.scales = p->n_kv_head * a.head_bytes;
    a.table_stride = p->table_stride;
    a.n_tok = (int)p->n_tok;
    a.n_seq = p->n_seq;
    a.n_head = p->n_head;
    a.n_kv = p->n_kv_head;
    a.group = p->n_head / p->n_kv_head;
    a.n_pages = p->max_pages > 0 ? (int)p->n_pages : 0;
    a.page_log2 = __builtin_ctz((unsigned)p->page_size);
    a.cap = p->max_pages * p->page_size;
    a.chunk = pl.chunk;
    a.n_split = pl.n_split;
    a.tiles = pl.tiles;
    a.c = p->scale * 1.4426950408889634f;
}
int run(const bonsai_p40_attn_paged_args * p, AttnArgs & a, const AttnLaunch & l, hipStream_t s) {
    if (p->kv_type == BONSAI_P40_Q8) return attn_q8_launch(a, l, s);
    const bool f32 = p->io_type == BONSAI_P40_F32;
    if (p->kv_type == BONSAI_P40_F16) return f32 ? launch_d<F16, 2>(l, a, s) : launch_d<F16, 1>(l, a, s);
    return f32 ? launch_d<BF16, 3>(l, a, s) : launch_d<BF16, 1>(l, a, s);
}

// ---- shared prefixes
int check_shared(const bonsai_p40_attn_shared_args * p) {
    if (!p || p->n_group < 0 || p->max_shared < 0) return 1;
    const int rc = check(&p->attn);
    return rc >= 0 ? rc : p->n_group > 0xffffff || (p->attn.n_tok + p->n_group) * (int64_t)p->attn.n_head >= 1 << 24 ? 1 : -1;
}
struct SharedPlan {
    Plan first, own;
};
SharedPlan plan_of(const bonsai_p40_attn_shared_args * p) {
    const int64_t cap = (int64_t)p->attn.max_pages * p->attn.page_size;
    const int64_t shared = p->max_shared > 0 && p->max_shared < cap ? p->max_shared : cap;
    // (own keys begin anywhere in 16; max_kv is not cut: a sequence of no group may have more of them than are left of the
    // table behind the longest prefix)
    const int64_t own = p->max_shared > 0 && p->attn.max_kv > shared ? p->attn.max_kv - shared + 15 : most_keys(&p->attn);
    return {plan_of(&p->attn, p->n_group, shared, SHARED_KEYS), plan_of(&p->attn, p->attn.n_seq, own < cap ? own : cap, OWN_KEYS)};
}

}  // namespace

extern "C" int64_t bonsai_p40_attn_paged_workspace_bytes(const bonsai_p40_attn_paged_args * p) {
    return check(p) == -1 ? part_bytes(p, plan_of(p, p->n_seq, most_keys(p)).n_split) : 0;
}

extern "C" int bonsai_p40_attn_paged(const bonsai_p40_attn_paged_args * p, bonsai_stream stream) {
    const int rc = check(p);
    if (rc >= 0) return rc;
    if (!pointers_ok(p)) return 1;
    Plan pl = plan_of(p, p->n_seq, most_keys(p));
    if (p->workspace == nullptr) pl.n_split = 1;
    else if (p->workspace_bytes < part_bytes(p, pl.n_split)) return 1;
    AttnArgs a;
    fill(a, p, pl);
    const AttnLaunch l = {pl.keys, pl.keys, false, pl.n_split > 1, p->io_type, p->head_dim};
    return run(p, a, l, (hipStream_t)stream);
}

extern "C" int64_t bonsai_p40_attn_shared_workspace_bytes(const bonsai_p40_attn_shared_args * p) {
    if (check_shared(p) != -1) return 0;
    if (p->n_group == 0) return bonsai_p40_attn_paged_workspace_bytes(&p->attn);
    const SharedPlan pl = plan_of(p);
    return part_bytes(&p->attn, pl.first.n_split + pl.own.n_split);
}

extern "C" int bonsai_p40_attn_shared(const bonsai_p40_attn_shared_args * p, bonsai_stream stream) {
    const int rc = check_shared(p);
    if (rc >= 0) return rc;
    if (p->n_group == 0) return bonsai_p40_attn_paged(&p->attn, stream);
    if (!pointers_ok(&p->attn) || pq2host::any_null(p->groups, p->shared, p->attn.workspace)) return 1;
    if (!aligned(p->groups, 4) || !aligned(p->shared, 4)) return 1;
    const SharedPlan pl = plan_of(p);
    if (p->attn.workspace_bytes < part_bytes(&p->attn, pl.first.n_split + pl.own.n_split)) return 1;
    AttnArgs a;
    fill(a, &p->attn, pl.own);
    a.groups = p->groups;
    a.shared = p->shared;
    a.n_group = p->n_group;
    a.chunk1 = pl.first.chunk;
    a.n_split1 = pl.first.n_split;
    a.tiles1 = pl.first.tiles;
    const AttnLaunch l = {pl.own.keys, pl.first.keys, true, true, p->attn.io_type, p->attn.head_dim};
    return run(&p->attn, a, l, (hipStream_t)stream);
}
