// kv_read.hip -- rows of a cache's pages read back by their slots
// (bonsai_p40_kv_read): what qk_norm_rope.hip wrote, as rows of fp32, f16 or bf16.
//
//   out_t = row of slot t,  d n for 8-bit pages
//
// It moves bytes: 1 or 2 in and 2 or 4 out an element.  A lane makes 16 bytes of
// output, a row's lanes are next to each other, and each lane has ROWS rows under way,
// as a slot, a row and its scale are a chain of two loads.  50001 rows of
// 4 heads of 256 from 8-bit pages (513 MB), inputs changing from call to call: 118 us with 4
// rows a lane, 122 with 2, 123 with 8; 4.4 TB/s, where a large copy reaches 5.4.  The same input
// again and again takes 88.
#include "host_state.h"
#include "launch_rules.h"
#include "mixer_device.h"

#include <type_traits>

using namespace mixer;

namespace {

struct ReadArgs {
    const uint8_t * pages[2];
    void * out[2];
    int64_t tok[2];                     // elements
    const int64_t * slots;
    int64_t n_slots, page_bytes, scales;
    int n_tok, n_kv, page_log2;
};

struct Q8 {
    typedef int8_t elem;
};

// PAST: stores past the caches
template <class TP, class TO, int D, bool PAST>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
    constexpr int E = 16 / sizeof(typename TO::elem), L = D / E, ROWS = 4;   // elements of a lane, lanes of a row
    constexpr bool BYTES = std::is_same<TP, Q8>::value;
    typedef typename TP::elem elem;
    typedef elem vec __attribute__((ext_vector_type(E)));
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const int e = threadIdx.x % L * E, t0 = blockIdx.x * (256 / L * ROWS) + threadIdx.x / L;
    const uint8_t * const pages = a.pages[which];
    int64_t slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) slot[i] = a.slots[min(t0 + i * (256 / L), a.n_tok - 1)];
    vec x[ROWS];
    float d[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        // (a slot outside reads the first one, which there is, and is not stored)
        const int64_t s = slot[i] >= 0 && slot[i] < a.n_slots ? slot[i] : 0, page = s >> a.page_log2;
        const int64_t row = ((int64_t)head << a.page_log2) + (s & ((1ll << a.page_log2) - 1));
        const uint8_t * const at = pages + page * a.page_bytes;
        x[i] = *reinterpret_cast<const vec *>(at + (row * D + e) * sizeof(elem));
        if (BYTES) d[i] = *reinterpret_cast<const float *>(at + a.scales + 4 * row);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int t = t0 + i * (256 / L);
        if (t >= a.n_tok || slot[i] < 0 || slot[i] >= a.n_slots) continue;
        float y[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if constexpr (BYTES) {
                y[j] = d[i] * (float)x[i][j];
                asm("" : "+v"(y[j]));                      // (the fp32 value is rounded, not the product)
            } else {
                y[j] = TP::to(x[i][j]);
            }
        typedef typename TO::elem row __attribute__((ext_vector_type(E)));
        row z;
#pragma unroll
        for (int j = 0; j < E; ++j) z[j] = TO::from(y[j]);
        row * const to = reinterpret_cast<row *>(reinterpret_cast<typename TO::elem *>(a.out[which]) + t * a.tok[which] + head * D + e);
        if (PAST) __builtin_nontemporal_store(z, to);
        else *to = z;
    }
}

template <class TP, class TO, int D>
int launch(const ReadArgs & a, hipStream_t s) {
    constexpr int size = sizeof(typename TO::elem), per = 256 / (D * size / 16) * 4;
    const dim3 grid((unsigned)((a.n_tok + per - 1) / per), (unsigned)(2 * a.n_kv));
    if (pq2::read_streams(2 * (int64_t)a.n_tok * a.n_kv * D * size))
        hipLaunchKernelGGL((kv_read_kernel<TP, TO, D, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_read_kernel<TP, TO, D, false>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}
template <class TP, class TO>
int launch_d(int d, const ReadArgs & a, hipStream_t s) {
    return d == 256 ? launch<TP, TO, 256>(a, s) : d == 128 ? launch<TP, TO, 128>(a, s) : launch<TP, TO, 64>(a, s);
}
template <class TP>
int launch_o(int out, int d, const ReadArgs & a, hipStream_t s) {
    return out == BONSAI_P40_F32 ? launch_d<TP, F32>(d, a, s) : out == BONSAI_P40_F16 ? launch_d<TP, F16>(d, a, s)
                                                                                     : launch_d<TP, BF16>(d, a, s);
}

}  // namespace

extern "C" int bonsai_p40_kv_read(const bonsai_p40_kv_read_args * p, bonsai_stream stream) {
    if (!p) return 1;
    const int d = p->head_dim;
    if (d != 64 && d != 128 && d != 256) return 1;
    if (p->n_kv_head < 1 || p->n_kv_head > 16384 || !is_type(p->out_type)) return 1;
    if ((!is_half(p->kv_type) && p->kv_type != BONSAI_P40_Q8) || !is_pow2(p->page_size) || p->page_size > 65536) return 1;
    if (p->n_pages < 0 || p->n_pages > (1ll << 40) || !page_stride_ok(p->kv_type, p->page_stride, p->n_kv_head, p->page_size, d)) return 1;
    const int per16 = 16 / type_bytes(p->out_type);
    if (p->k_tok < (int64_t)p->n_kv_head * d || p->k_tok % per16 != 0) return 1;
    if (p->v_tok < (int64_t)p->n_kv_head * d || p->v_tok % per16 != 0) return 1;
    if (p->n_tok <= 0 || p->n_pages == 0) return 0;
    if (p->n_tok > 0x7fffffff / 2 || p->n_tok * (int64_t)p->n_kv_head * d > 1ll << 34) return 1;   // a grid has fewer than 2^32 threads
    if (pq2host::any_null(p->k_pages, p->v_pages, p->slots, p->k_out, p->v_out)) return 1;
    if (!aligned(p->k_pages, 16) || !aligned(p->v_pages, 16) || !aligned(p->k_out, 16) || !aligned(p->v_out, 16) || !aligned(p->slots, 8))
        return 1;
    const int el = p->kv_type == BONSAI_P40_Q8 ? 1 : 2;
    ReadArgs a;
    a.pages[0] = reinterpret_cast<const uint8_t *>(p->k_pages);
    a.pages[1] = reinterpret_cast<const uint8_t *>(p->v_pages);
    a.out[0] = p->k_out;
    a.out[1] = p->v_out;
    a.tok[0] = p->k_tok;
    a.tok[1] = p->v_tok;
    a.slots = p->slots;
    a.page_log2 = __builtin_ctz((unsigned)p->page_size);
    a.n_slots = p->n_pages << a.page_log2;
    a.page_bytes = p->page_stride * el;
    a.scales = (int64_t)p->n_kv_head * p->page_size * d;
    a.n_tok = (int)p->n_tok;
    a.n_kv = p->n_kv_head;
    const hipStream_t s = (hipStream_t)stream;
    return p->kv_type == BONSAI_P40_F16 ? launch_o<F16>(p->out_type, d, a, s) : p->kv_type == BONSAI_P40_BF16 ? launch_o<BF16>(p->out_type, d, a, s)
                                                                                                         : launch_o<Q8>(p->out_type, d, a, s);
}
