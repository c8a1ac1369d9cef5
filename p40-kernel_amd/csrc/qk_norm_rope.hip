// qk_norm_rope.hip -- between the q/k/v projections and attention: RMSNorm of
// every query and key head, position rotation, and the append of keys and
// values to the pages of the cache, in one launch (bonsai_p40_qk_norm_rope).
//
//   y = x / sqrt(mean(x^2) + eps) * w                       per head row
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s),  c, s = cos, sin(pos f_i)
//
// It moves bytes and little else: 4 in and 2 or 4 out an element.  A workgroup
// takes one head row of TT tokens (4, 16 or 32: rope_tile); the angles of those tokens are computed once
// into LDS.  An angle is pos * f / 2 pi in fp64, reduced to half a turn there:
// in fp32 a position of 1e6 would leave it 4 bits.
//   Rows (one per token): a wave reads a token's head row from memory.
//   Columns (one row per feature, as bonsai_p40_gemm writes): the tile of
// head_dim features x TT tokens goes through LDS, a row's 16-byte units permuted by
// its token: they are read 16 bytes a lane, and written with two lanes on a bank.
// (Padded rows would leave room for 3 workgroups a CU of 32 x 256, not 4: 30.1
// us for 26.6, 2048 tokens of 24 + 4 + 4 heads, f16: 101 MB, 3.8 TB/s.)  All of a
// tile's loads are asked for at once.
#include "host_state.h"
#include "launch_rules.h"
#include "mixer_device.h"
#include "pq2_device.h"

using namespace mixer;

namespace {

struct QkvArgs {
    const float * x[3];                 // q, k, v
    int64_t tok[3], head[3], el[3];     // strides in floats
    const float * w[3];                 // norm weights or NULL
    const int32_t * pos;
    const double * inv_freq;
    const int64_t * slots;
    void * q_out;
    int64_t q_out_tok;
    void * pages[2];                    // k, v
    int64_t page_stride, n_slots;
    float eps;
    int n_tok, n_head, n_kv, half, interleaved, page_log2, tt, vec;
};

template <int D, class TQ, class TC>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkvArgs a) {
    constexpr int E = D / 64;           // consecutive elements of a lane
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int row = blockIdx.y;
    const int kind = row < a.n_head ? 0 : row < a.n_head + a.n_kv ? 1 : 2;
    row -= kind == 0 ? 0 : a.n_head + (kind - 1) * a.n_kv;
    const int t0 = blockIdx.x * a.tt, nt = min(a.tt, a.n_tok - t0);
    const float * const x = a.x[kind] + (int64_t)row * a.head[kind];
    const int64_t ts = a.tok[kind], es = a.el[kind];
    const bool columns = es != 1;
    float * const tile = lds;                                            // [tt][D] where columns, element e at e ^ place(t)
    float2 * const turn = reinterpret_cast<float2 *>(lds + (columns ? a.tt * D : 0));         // [tt][half]
    auto place = [](int t) { return 4 * (t & 15); };

    if (columns) {
        // the tokens of a feature are one run of up to 128 bytes: half a wave each
        const int sub = threadIdx.x & 31;
        if (sub < nt) {
            const float * const c = x + (int64_t)(t0 + sub) * ts + (int64_t)(threadIdx.x >> 5) * es;
            float * const to = tile + sub * D;
            float v[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) v[i] = c[(int64_t)(8 * i) * es];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float * const at = to + ((8 * i + (threadIdx.x >> 5)) ^ place(sub));
#pragma unroll
                for (int j = 0; j < D / 64; ++j) at[64 * j] = v[8 * j + i];
            }
        }
    }
    if (kind < 2) {
        for (int i = threadIdx.x; i < nt * a.half; i += 256) {
            const int t = i / a.half, f = i - t * a.half;
            const double rev = (double)a.pos[t0 + t] * a.inv_freq[f] * 0.15915494309189535;
            const float r = (float)(rev - rint(rev));
            float sn, cs;
            sincospif(2.0f * r, &sn, &cs);
            turn[i] = make_float2(cs, sn);
        }
    }
    __syncthreads();

    float w[E];
#pragma unroll
    for (int j = 0; j < E; ++j) w[j] = 1.0f;
    const bool norm = kind < 2 && a.w[kind] != nullptr;
    if (norm)
#pragma unroll
        for (int j = 0; j < E; ++j) w[j] = a.w[kind][lane * E + j];

    auto load = [&](int t, float (&v)[E]) {
        if (columns) {
            load_row<F32>(tile + t * D + ((lane * E) ^ place(t)), v);
        } else {
            const float * const r = x + (int64_t)(t0 + t) * ts + lane * E;
            if (a.vec) load_row<F32>(r, v);
            else
#pragma unroll
                for (int j = 0; j < E; ++j) v[j] = r[j];
        }
    };
    // 4 rows at a time, side by side: one alone is a chain of waits (a reduction, the partner's elements)
    const float2 * const angles = turn;
    constexpr int B = 4;
    for (int tb = wave; tb < nt; tb += 4 * B) {
        float v[B][E];
#pragma unroll
        for (int k = 0; k < B; ++k) load(min(tb + 4 * k, nt - 1), v[k]);
        if (norm) {
            float ss[B];
#pragma unroll
            for (int k = 0; k < B; ++k) {
                ss[k] = 0.0f;
#pragma unroll
                for (int j = 0; j < E; ++j) ss[k] = fmaf(v[k][j], v[k][j], ss[k]);
            }
#pragma unroll
            for (int k = 0; k < B; ++k) ss[k] = pq2::wave_sum_to_lane63(ss[k]);
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const float sum = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ss[k]), 63));
                const float s = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
                for (int j = 0; j < E; ++j) v[k][j] = v[k][j] * s * w[j];
            }
        }
        if (kind < 2 && a.half > 0) {
            // the partner is half elements away, a whole number of lanes, or the next element
            const int d = a.half / E, src = (lane < d ? lane + d : lane - d) & 63;
            const bool in = lane * E < 2 * a.half;
            float o[B][E];
#pragma unroll
            for (int k = 0; k < B; ++k)
#pragma unroll
                for (int j = 0; j < E; ++j)
                    o[k][j] = !a.interleaved ? __shfl(v[k][j], src) : E == 1 ? __shfl_xor(v[k][j], 1) : v[k][j ^ (E > 1)];
            if (in) {
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const float2 * const tr = angles + min(tb + 4 * k, nt - 1) * a.half;
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const int e = lane * E + j;
                        const bool second = a.interleaved ? (e & 1) : e >= a.half;
                        const float2 cs = tr[a.interleaved ? e >> 1 : second ? e - a.half : e];
                        v[k][j] = fmaf(second ? o[k][j] : -o[k][j], cs.y, v[k][j] * cs.x);
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int t = tb + 4 * k;
            if (t >= nt) break;
            if (kind == 0) {
                store_row<TQ>(reinterpret_cast<typename TQ::elem *>(a.q_out) + (int64_t)(t0 + t) * a.q_out_tok +
                                  (int64_t)row * D + lane * E, v[k]);
            } else {
                const int64_t slot = a.slots[t0 + t];
                if (slot >= 0 && slot < a.n_slots) {
                    const int64_t page = slot >> a.page_log2, off = slot & ((1ll << a.page_log2) - 1);
                    store_row<TC>(reinterpret_cast<typename TC::elem *>(a.pages[kind - 1]) + page * a.page_stride +
                                      (((int64_t)row << a.page_log2) + off) * D + lane * E, v[k]);
                }
            }
        }
    }
}

template <int D, class TQ, class TC>
void launch(const QkvArgs & a, dim3 grid, size_t bytes, hipStream_t s) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<D, TQ, TC>), grid, dim3(256), bytes, s, a);
}
template <int D, class TQ>
void launch_c(int kv, const QkvArgs & a, dim3 grid, size_t bytes, hipStream_t s) {
    if (kv == BONSAI_P40_F16) launch<D, TQ, F16>(a, grid, bytes, s);
    else launch<D, TQ, BF16>(a, grid, bytes, s);
}
template <int D>
void launch_q(int q, int kv, const QkvArgs & a, dim3 grid, size_t bytes, hipStream_t s) {
    if (q == BONSAI_P40_F32) launch_c<D, F32>(kv, a, grid, bytes, s);
    else if (q == BONSAI_P40_F16) launch_c<D, F16>(kv, a, grid, bytes, s);
    else launch_c<D, BF16>(kv, a, grid, bytes, s);
}

}  // namespace

extern "C" int bonsai_p40_qk_norm_rope(const bonsai_p40_qk_norm_rope_args * p, bonsai_stream stream) {
    if (!p) return 1;
    const int d = p->head_dim;
    if (d != 64 && d != 128 && d != 256) return 1;
    if (p->n_head < 1 || p->n_kv_head < 1 || p->n_head > 16384 || p->n_kv_head > 16384) return 1;
    if (p->n_rot < 0 || p->n_rot > d || p->n_rot % 8 != 0) return 1;
    if (!is_type(p->q_type) || !is_half(p->kv_type) || !is_pow2(p->page_size) || p->page_size > 65536) return 1;
    if (p->n_pages < 0 || p->n_pages > (1ll << 40) || p->page_stride < (int64_t)p->n_kv_head * p->page_size * d || p->page_stride % 8 != 0) return 1;
    if (p->q_out_tok < (int64_t)p->n_head * d || p->q_out_tok % (16 / type_bytes(p->q_type)) != 0) return 1;
    if (p->n_tok <= 0) return 0;
    if (p->n_tok > 0x7fffffff / 64) return 1;
    if (pq2host::any_null(p->q, p->k, p->v, p->slots, p->q_out, p->k_pages, p->v_pages)) return 1;
    if (p->n_rot > 0 && pq2host::any_null(p->pos, p->inv_freq)) return 1;
    if (!aligned(p->q_out, 16) || !aligned(p->k_pages, 16) || !aligned(p->v_pages, 16)) return 1;
    if (!aligned(p->q_norm, 4) || !aligned(p->k_norm, 4) || !aligned(p->pos, 4) || !aligned(p->inv_freq, 8) ||
        !aligned(p->slots, 8))
        return 1;
    QkvArgs a;
    const float * const x[3] = {p->q, p->k, p->v};
    const int64_t st[3][3] = {{p->q_tok, p->q_head, p->q_el}, {p->k_tok, p->k_head, p->k_el}, {p->v_tok, p->v_head, p->v_el}};
    bool columns = false;
    a.vec = 1;
    for (int i = 0; i < 3; ++i) {
        if (st[i][2] != 1 && (st[i][0] != 1 && p->n_tok > 1)) return 1;   // features or tokens are consecutive
        a.x[i] = x[i];
        a.tok[i] = st[i][0];
        a.head[i] = st[i][1];
        a.el[i] = st[i][2];
        if (!aligned(x[i], 4)) return 1;
        if (st[i][2] != 1) columns = true;
        else if (!aligned(x[i], 16) || st[i][0] % 4 != 0 || st[i][1] % 4 != 0) a.vec = 0;
    }
    a.w[0] = p->q_norm;
    a.w[1] = p->k_norm;
    a.w[2] = nullptr;
    a.pos = p->pos;
    a.inv_freq = p->inv_freq;
    a.slots = p->slots;
    a.q_out = p->q_out;
    a.q_out_tok = p->q_out_tok;
    a.pages[0] = p->k_pages;
    a.pages[1] = p->v_pages;
    a.page_stride = p->page_stride;
    a.page_log2 = __builtin_ctz((unsigned)p->page_size);
    a.n_slots = p->n_pages << a.page_log2;
    a.eps = p->eps;
    a.n_tok = (int)p->n_tok;
    a.n_head = p->n_head;
    a.n_kv = p->n_kv_head;
    a.half = p->n_rot / 2;
    a.interleaved = p->interleaved != 0;
    a.tt = pq2::rope_tile(columns, p->n_tok);
    auto lds = [&](int tt) { return (columns ? (size_t)tt * d * 4 : 0) + (size_t)tt * a.half * 8; };
    // 3 workgroups to a CU at least: 2048 tokens of 256 columns, us, 16 / 32: 256 of them rotated 38.8 / 42.9, 128 34.9 / 32.1
    if (lds(a.tt) > 53 * 1024) a.tt = 16;
    const size_t bytes = lds(a.tt);
    const dim3 grid((unsigned)((p->n_tok + a.tt - 1) / a.tt), (unsigned)(p->n_head + 2 * p->n_kv_head));
    const hipStream_t s = (hipStream_t)stream;
    if (d == 256) launch_q<256>(p->q_type, p->kv_type, a, grid, bytes, s);
    else if (d == 128) launch_q<128>(p->q_type, p->kv_type, a, grid, bytes, s);
    else launch_q<64>(p->q_type, p->kv_type, a, grid, bytes, s);
    return (int)hipGetLastError();
}
