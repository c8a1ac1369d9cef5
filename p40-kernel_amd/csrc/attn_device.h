// attn_device.h -- what the kernels of attention over pages have in common
// (attn_paged.hip: 16-bit pages, attn_q8.hip: 8-bit ones): their arguments, whose
// rows and keys a workgroup takes, and the join of a row's parts.
//
// Batches that share a prefix (bonsai_p40_attn_shared) go through the same kernels
// in two phases: the rows of a whole group, as if they were one sequence's, over the
// group's shared keys, all of which they see; and each sequence's rows over its own
// keys, which begin behind the shared ones.  Both leave parts (sums with the maximum
// that they are relative to), and the join adds them as it adds those of a split.
#pragma once

#include "launch_rules.h"
#include "mixer_device.h"

#include <math.h>

namespace mixer {

struct AttnArgs {
    const void * q;
    void * out;
    const uint8_t * k, * v;
    const int32_t * table, * starts, * kv_len;
    float * part;                       // [part][row][D] then [part][row] (m, l)
    int64_t q_tok, out_tok;             // elements
    int64_t page_bytes, head_bytes;
    int64_t table_stride;
    int n_tok, n_seq, n_head, n_kv, group;
    int n_pages, page_log2, cap;        // cap: keys the table can name
    int chunk, n_split, tiles;
    float c;                            // scale * log2(e)
    // 8-bit pages: where a page's scales begin
    int64_t scales;
    // shared prefixes: the groups, the shared keys of each, and their phase, whose blocks come first
    const int32_t * groups, * shared;
    int n_group;
    int chunk1, n_split1, tiles1;
    unsigned blocks1;
};

// The arguments once more, from the kernel's own memory of them: what is read through this is loaded where it is used
typedef const __attribute__((address_space(4))) AttnArgs LateArgs;
__device__ __forceinline__ LateArgs * late_args() {
    uintptr_t p = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return (LateArgs *)p;
}

template <bool LATE>
__device__ __forceinline__ auto args_of(const AttnArgs & a) {
    if constexpr (LATE) return late_args();
    else return &a;
}

// 1 / l; 0 where no key was seen, NaN where the score of every key that was is -inf
__device__ __forceinline__ float over(float m, float l) { return m == -INFINITY ? 0.0f : l != 0.0f ? 1.0f / l : NAN; }

// The shared keys of sequence seq's group; -1: it is in none.  For whole waves.  only: the one group there is, asked
// for beside what seq follows from
struct OneGroup {
    int first, next, keys;
};
__device__ __forceinline__ OneGroup one_group(const AttnArgs & a) {
    if (a.n_group == 1) return OneGroup{sload(a.groups, 0), sload(a.groups, 1), sload(a.shared, 0)};
    return OneGroup{0, 0, 0};
}
__device__ __forceinline__ int shared_of(const AttnArgs & a, const OneGroup & only, int seq) {
    if (a.n_group == 1) return seq >= only.first && seq < only.next ? iclamp(only.keys, 0, a.cap) : -1;
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < a.n_group; g0 += 64) {
        const int g = g0 + lane;
        int b = 0, e = 0, n = 0;
        if (g < a.n_group) {
            b = a.groups[g];
            e = a.groups[g + 1];
            n = a.shared[g];
        }
        const uint64_t hit = __ballot(seq >= b && seq < e);
        if (hit) return iclamp(__builtin_amdgcn_readlane(n, __builtin_ctzll(hit)), 0, a.cap);
    }
    return -1;
}

// find_tile for the rows of whole groups: seq is a group's first sequence, extra its shared keys.  A wave takes
// 64 groups a step
template <int BM>
__device__ __forceinline__ Tile find_group_tile(const AttnArgs & a, int tile) {
    if (a.n_group == 1) {               // no search
        const int first = iclamp(sload(a.groups, 0), 0, a.n_seq), next = iclamp(sload(a.groups, 1), 0, a.n_seq), x = sload(a.shared, 0);
        const int b = iclamp(sload(a.starts, first), 0, a.n_tok), n = max(iclamp(sload(a.starts, next), 0, a.n_tok) - b, 0);
        const int tiles = (int)(((int64_t)n * a.group + BM - 1) / BM);
        return Tile{tile < tiles ? first : -1, tile, b, n, x};
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int g0 = 0; g0 < a.n_group; g0 += 64) {
        const int g = g0 + lane;
        int b = 0, n = 0, x = 0, first = 0;
        if (g < a.n_group) {
            first = iclamp(a.groups[g], 0, a.n_seq);
            x = a.shared[g];
            const int next = iclamp(a.groups[g + 1], 0, a.n_seq);
            b = iclamp(a.starts[first], 0, a.n_tok);
            n = max(iclamp(a.starts[next], 0, a.n_tok) - b, 0);
        }
        const int own = (int)(((int64_t)n * a.group + BM - 1) / BM);
        int sum = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const uint64_t hit = __ballot(base + sum > tile);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            Tile t;
            t.seq = __builtin_amdgcn_readlane(first, l);
            t.index = tile - (base + __builtin_amdgcn_readlane(sum - own, l));
            t.first = __builtin_amdgcn_readlane(b, l);
            t.count = __builtin_amdgcn_readlane(n, l);
            t.extra = __builtin_amdgcn_readlane(x, l);
            return t;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return Tile{-1, 0, 0, 0, 0};
}

// A workgroup's rows and keys.  A sequence's own keys begin at lo, their parts at the 16 keys that hold it
struct AttnPlace {
    bool pre;                           // of the shared prefixes
    int kvh, split, tile;
};
template <bool SHARED, class Args>
__device__ __forceinline__ AttnPlace attn_place(Args * a) {
    AttnPlace p;
    p.pre = SHARED && blockIdx.x < a->blocks1;
    // (unsigned: these divisions are ahead of the first load)
    const unsigned block = SHARED && !p.pre ? blockIdx.x - a->blocks1 : blockIdx.x, n_kv = a->n_kv;
    const unsigned tiles = SHARED && p.pre ? a->tiles1 : a->tiles;
    // heads vary fastest: a head's tiles meet on the same XCDs, and then in their L2, as those that run at the
    // same time have the same keys; the last tiles, which see the most, start first
    p.kvh = (int)(block % n_kv);
    const unsigned rest = block / n_kv;
    p.split = (int)(rest / tiles);
    p.tile = (int)(tiles - 1 - rest % tiles);
    return p;
}
// its place among the parts of a row
template <bool SHARED, class Args>
__device__ __forceinline__ int attn_part(Args * a, const AttnPlace & p) {
    return SHARED && !p.pre ? a->n_split1 + p.split : p.split;
}
// Of kv keys, how many token tok sees.  (Without SHARED, where its own is one of them, nothing can overflow)
template <bool SHARED>
__device__ __forceinline__ int keys_seen(int before, int kv, int tok) {
    return SHARED ? pq2::attn_seen(before, kv, tok) : iclamp(before + tok + 1, 0, kv);
}
struct AttnWork {
    Tile tl;
    int lo;
    int kv, before, nk, k0, k1;         // keys k0 .. k1 of nk; of kv a row sees keys_seen
};
// false: there is nothing to do
template <int BM, bool SHARED>
__device__ __forceinline__ bool attn_work(const AttnArgs & a, const AttnPlace & p, AttnWork & w) {
    OneGroup only = {0, 0, 0};
    if (SHARED && !p.pre) only = one_group(a);
    w.tl = SHARED && p.pre ? find_group_tile<BM>(a, p.tile)
                           : find_tile<BM>(a.starts, a.kv_len, a.n_seq, a.n_tok, a.group, p.tile);
    if (w.tl.seq < 0) return false;
    w.lo = SHARED && !p.pre ? max(shared_of(a, only, w.tl.seq), 0) : 0;
    const int rows = w.tl.count * a.group, last = min((w.tl.index + 1) * BM, rows) - 1;
    w.kv = iclamp(w.tl.extra, 0, a.cap);
    w.before = SHARED && p.pre ? w.kv : w.kv - w.tl.count;     // (pre: every row sees all of them)
    // (readfirstlane: the same in all lanes, which the compiler does not see through the division)
    w.nk = a.n_pages > 0 ? __builtin_amdgcn_readfirstlane(keys_seen<SHARED>(w.before, w.kv, last / a.group)) : 0;
    if (SHARED) {
        // (64 bits: where the host knows no lengths, the last part may begin anywhere)
        const int chunk = p.pre ? a.chunk1 : a.chunk, n_split = p.pre ? a.n_split1 : a.n_split;
        const int64_t k0 = (int64_t)(w.lo & ~15) + (int64_t)p.split * chunk;
        w.k0 = (int)min(k0, (int64_t)0x7fffffff);
        w.k1 = p.split == n_split - 1 ? w.nk : (int)min((int64_t)w.nk, k0 + chunk);
    } else {
        w.k0 = p.split * a.chunk;
        w.k1 = p.split == a.n_split - 1 ? w.nk : min(w.nk, w.k0 + a.chunk);
    }
    return p.split == 0 || w.k0 < w.nk;                    // the join counts the parts
}
// ... of them, for nk keys, the first of them in the 16 that hold lo
__device__ __forceinline__ int attn_parts(int nk, int lo, int chunk, int n_split) {
    const int keys = max(nk - (lo & ~15), 0);
    return iclamp((int)(((uint32_t)keys + (uint32_t)chunk - 1) / (uint32_t)chunk), 1, n_split);
}

}  // namespace mixer

namespace {

using namespace mixer;

// The parts of every row, by WR waves.  Their number follows from the keys the
// row's tile saw, as in attn_work; the largest m is looked for among all that
// there could be while the lengths are on their way.
template <class TO, int D, int WR, bool SHARED>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int bm) {
    constexpr int E = D / 64, AHEAD = 8;
    __shared__ float sum[4][D + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % WR;
    const int64_t all_rows = (int64_t)a.n_tok * a.n_head, row = (int64_t)blockIdx.x * (4 / WR) + wave / WR;
    if (row >= all_rows) return;
    const int tok = (int)(row / a.n_head), head = (int)(row - (int64_t)tok * a.n_head);
    const int first_parts = SHARED ? a.n_split1 : 0, n_part = first_parts + a.n_split;
    const float2 * const ml = reinterpret_cast<const float2 *>(a.part + (int64_t)n_part * all_rows * D) + row;
    float own = -INFINITY;
    if (lane < n_part) own = ml[lane * all_rows].x;
    // (4 waves: the first parts, too; those behind the last are not written, and not used)
    float v[AHEAD][E];
    float2 e[AHEAD];
    // part i: the parts of a shared prefix, which are n1, come first, the others behind the place of the last there could be
    auto load = [&](int k, int64_t i) __attribute__((always_inline)) {
        e[k] = ml[i * all_rows];
        load_row<F32>(a.part + (i * all_rows + row) * D + lane * E, v[k]);
    };
    OneGroup only = {0, 0, 0};
    constexpr int OWN = SHARED ? AHEAD - 1 : 0;            // SHARED: the last of the first loads is of the own keys' parts
    if (SHARED) {
        only = one_group(a);
#pragma unroll
        for (int k = 0; k < OWN; ++k) load(k, min(w + k * WR, first_parts - 1));
        load(OWN, first_parts + min(w, a.n_split - 1));
    } else if (WR > 1) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) load(k, min(w + k * WR, a.n_split - 1));
    }
    // the sequence of this token
    int seq = -1, first = 0, count = 0, kv = 0;
    for (int s0 = 0; s0 < a.n_seq && seq < 0; s0 += 64) {
        const int s = s0 + lane;
        int b = 0, e = 0, len = 0;
        if (s < a.n_seq) {
            b = iclamp(a.starts[s], 0, a.n_tok);
            e = iclamp(a.starts[s + 1], 0, a.n_tok);
            len = iclamp(a.kv_len[s], 0, a.cap);
        }
        const uint64_t hit = __ballot(tok >= b && tok < e);
        if (hit) {
            const int k = __builtin_ctzll(hit);
            seq = s0 + k;
            first = __builtin_amdgcn_readlane(b, k);
            count = __builtin_amdgcn_readlane(e, k) - first;
            kv = __builtin_amdgcn_readlane(len, k);
        }
    }
    if (seq < 0) return;                                   // a row behind the last sequence
    int lo = 0, n1 = 0;
    if (SHARED) {
        const int s = shared_of(a, only, seq);
        lo = max(s, 0);
        if (s >= 0) n1 = attn_parts(a.n_pages > 0 ? s : 0, 0, a.chunk1, a.n_split1);
    }
    const int r = (tok - first) * a.group + head % a.group;
    const int last = min(r / bm * bm + bm, count * a.group) - 1;
    const int nk = a.n_pages > 0 ? iclamp(kv - count + last / a.group + 1, 0, kv) : 0;
    const int n = attn_parts(nk, lo, a.chunk, a.n_split);
    auto there = [&](int i) { return SHARED ? i < n1 || (i >= first_parts && i < first_parts + n) : i < n; };
    float mm = there(lane) ? own : -INFINITY;
    for (int i = 64 + lane; i < (SHARED ? n_part : n); i += 64)
        if (!SHARED || there(i)) mm = fmaxf(mm, ml[i * all_rows].x);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float x[E] = {}, l = 0.0f;
    auto add = [&](int k) __attribute__((always_inline)) {
        const float wt = __builtin_amdgcn_exp2f(e[k].x - ref);
        l = fmaf(e[k].y, wt, l);
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = fmaf(v[k][j], wt, x[j]);
    };
    // parts base + from, from + WR, .. of base + count
    auto rest = [&](int base, int from, int count) __attribute__((always_inline)) {
        for (int i0 = from; i0 < count; i0 += WR * AHEAD) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) load(k, base + min(i0 + k * WR, count - 1));
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (i0 + k * WR < count) add(k);
        }
    };
    if (SHARED) {
#pragma unroll
        for (int k = 0; k < OWN; ++k)
            if (w + k * WR < n1) add(k);
        if (w < n) add(OWN);
        rest(0, w + OWN * WR, n1);
        rest(first_parts, w + WR, n);
    } else {
        if (WR > 1) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (w + k * WR < n) add(k);
        }
        rest(0, WR > 1 ? w + WR * AHEAD : w, n);
    }
    if constexpr (WR > 1) {
#pragma unroll
        for (int j = 0; j < E; ++j) sum[wave][lane * E + j] = x[j];
        if (lane == 0) sum[wave][D] = l;
        __syncthreads();                                   // (WR = 4: one row a workgroup, all waves are here)
        if (w) return;
        for (int k = 1; k < WR; ++k) {
            l += sum[k][D];
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] += sum[k][lane * E + j];
        }
    }
    const float inv = over(mm, l);
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] *= inv;
    store_row<TO>(reinterpret_cast<typename TO::elem *>(a.out) + (int64_t)tok * a.out_tok + (int64_t)head * D + lane * E, x);
}

template <class TO, int D, bool SHARED>
inline int launch_join(const AttnArgs & a, int bm, hipStream_t s) {
    const int64_t rows = (int64_t)a.n_tok * a.n_head;
    if (pq2::attn_join_wide(a.n_split + (SHARED ? a.n_split1 : 0)))
        hipLaunchKernelGGL((attn_join_kernel<TO, D, 4, SHARED>), dim3((unsigned)rows), dim3(256), 0, s, a, bm);
    else hipLaunchKernelGGL((attn_join_kernel<TO, D, 1, SHARED>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, bm);
    return (int)hipGetLastError();
}

}  // namespace

namespace mixer {

// ---- host: the entry points of attn_paged.hip hand 8-bit pages to attn_q8.hip
// keys, keys1: the waves split the keys (else the rows); parts: a.part is used
struct AttnLaunch {
    bool keys, keys1, shared, parts;
    int io_type, head_dim;
};
int attn_q8_launch(AttnArgs & a, const AttnLaunch & l, hipStream_t s);

}  // namespace mixer
