// mixer_device.h -- element types of the token mixers (qk_norm_rope.hip,
// attn_paged.hip, gdn.hip): fp32, f16 and bf16 rows, computed on in fp32.
// Stores round to nearest, ties to even, once.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/bonsai_p40.h"

namespace mixer {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

// storage types: each converts to and from fp32
struct F32 {
    typedef float elem;
    static __device__ __forceinline__ float to(elem v) { return v; }
    static __device__ __forceinline__ elem from(float v) { return v; }
};
struct F16 {
    typedef _Float16 elem;
    typedef v8h frag;
    static constexpr uint32_t EXP = 0x7c00;     // exponent bits: all set in infinities and NaN
    static __device__ __forceinline__ float to(elem v) { return (float)v; }
    static __device__ __forceinline__ elem from(float v) { return (elem)v; }
};
struct BF16 {
    typedef __bf16 elem;
    typedef v8b frag;
    static constexpr uint32_t EXP = 0x7f80;
    static __device__ __forceinline__ float to(elem v) { return (float)v; }
    static __device__ __forceinline__ elem from(float v) { return (elem)v; }
};

// E consecutive elements as fp32; the pointer is aligned to E elements
template <class T, int E>
__device__ __forceinline__ void load_row(const typename T::elem * p, float (&v)[E]) {
    typedef typename T::elem vec __attribute__((ext_vector_type(E)));
    const vec x = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = T::to(x[i]);
}
template <class T, int E>
__device__ __forceinline__ void store_row(typename T::elem * p, const float (&v)[E]) {
    typedef typename T::elem vec __attribute__((ext_vector_type(E)));
    vec x;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = T::from(v[i]);
    *reinterpret_cast<vec *>(p) = x;
}

__device__ __forceinline__ int iclamp(int v, int lo, int hi) { return min(max(v, lo), hi); }
// a uniform load through the scalar cache
__device__ __forceinline__ int sload(const int32_t * p, int64_t i) {
    typedef const __attribute__((address_space(4))) int32_t cint;
    return *(cint *)(uintptr_t)(p + i);
}
// 16 bytes a lane from a buffer (uniform base, a lane's offset, a constant one) to
// LDS: dst is the wave's, lane l lands at dst + 16 l.  Through the buffer path, as
// beside the global one (which counts as a flat access) the compiler's waits for
// LDS reads no longer count, but wait for all.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t * base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), (short)0, bytes, 0x00020000);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t from, uint8_t * dst, int off, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void *)dst, 16, off, soff, 0, 0);
}
// BOTH bytes further on either side (the instruction's own offset counts for both)
template <int BOTH>
__device__ __forceinline__ void dma16_at(__amdgpu_buffer_rsrc_t from, uint8_t * dst, int off, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void *)dst, 16, off, soff, BOTH, 0);
}

// Which sequence a tile of up to BM rows (per_tok of them a token) belongs to;
// the tiles of sequence s follow those of s - 1.  starts: n_seq + 1 entries, cut
// to 0 .. n_tok.  seq is -1 behind the last tile.  For whole waves.
struct Tile {
    int seq, index, first, count;       // sequence, its tile, its first token, its tokens
    int extra;                          // its entry of `more` (NULL: 0), read beside starts
};
template <int BM>
__device__ __forceinline__ Tile find_tile(const int32_t * starts, const int32_t * more, int n_seq, int n_tok, int per_tok,
                                          int tile) {
    if (n_seq == 1) {                   // no search, two waits less
        const int b = iclamp(sload(starts, 0), 0, n_tok), n = max(iclamp(sload(starts, 1), 0, n_tok) - b, 0);
        const int tiles = (int)(((int64_t)n * per_tok + BM - 1) / BM);
        return Tile{tile < tiles ? 0 : -1, tile, b, n, more ? sload(more, 0) : 0};
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < n_seq; s0 += 64) {
        const int s = s0 + lane;
        int b = 0, n = 0, x = 0;
        if (s < n_seq) {
            b = iclamp(starts[s], 0, n_tok);
            n = max(iclamp(starts[s + 1], 0, n_tok) - b, 0);
            if (more) x = more[s];
        }
        const int own = (int)(((int64_t)n * per_tok + BM - 1) / BM);
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
            t.seq = s0 + l;
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

inline int type_bytes(int t) { return t == BONSAI_P40_F32 ? 4 : 2; }
inline bool is_type(int t) { return t == BONSAI_P40_F32 || t == BONSAI_P40_F16 || t == BONSAI_P40_BF16; }
inline bool is_half(int t) { return t == BONSAI_P40_F16 || t == BONSAI_P40_BF16; }
inline bool is_pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }
inline bool aligned(const void * p, unsigned a) { return ((uintptr_t)p & (a - 1)) == 0; }

}  // namespace mixer
