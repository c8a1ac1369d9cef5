// gdn.hip -- the gated delta rule of the linear-attention layers
// (bonsai_p40_gdn).  Token by token, for a state S of K x V fp32 of each value head:
//
//   S <- e^g S,   u = beta (v - S^T k),   S <- S + k u^T,   o = scale S^T q.
//
// Few tokens: gdn_step_kernel.  A wave keeps 16 columns of S in registers (they
// never meet the other columns) and runs through the tokens; with a = S^T k and
// b = S^T q of the old state, o = e^g b + (q.k) u, so that one reduction serves
// both.  Bound by the state's bytes, read and written once.
//
// Many: chunks of 64 tokens.  With G the sums of g inside a chunk and S0 its first state,
//   L_ij = beta_i (k_i.k_j) e^(Gi - Gj) (j < i),   T = (I + L)^-1 diag(beta),
//   U = T (v - e^G * (K S0)),   o = scale (e^G * (Q S0) + tril((q_i.k_j) e^(Gi - Gj)) U),
//   S = e^Gc S0 + (K e^(Gc - G))^T U,
// which are matrix products.  gdn_prep_kernel makes what does not depend on S
// (T, the masked QK^T, K, Q and K^T) for all chunks at once, gdn_scan_kernel goes
// through the chunks.
//   The outputs are fp32's, so the products are, too: each operand is split into
// two f16 terms and the products hi hi, hi lo and lo hi run on v_mfma_f32_16x16x32_f16,
// the three of them at 5 times the rate of fp32's own matrix instructions.  Rows of the
// left and columns of the right operand are scaled by powers of two so that their largest
// is 2^14 to 2^15, near f16's end: the terms hold 22 bits of what is 2^-18 of that
// and more, and are off by up to 2^-40 of it below.  (With the largest at 1 the 22 bits
// would end at 2^-4: a token's values 2^10 above the others' cost the tokens before it
// 3.0e-5 of their rows, for 4.2e-7; 2^20 3.2e-2 for 1.8e-6.)
//   G is summed in fp64 and kept as two floats: after a strong decay the differences of
// fp32 sums would have no digits left.
//   In the scan a wave has 16 columns of S, R and U to itself: a result tile
// (lane: column, 4 rows 4 g .. 4 g + 3) is the next product's right operand as it
// stands, if the left one lists its contraction as 4 g + j, 16 + 4 g + j (j < 4).
// So nothing of the chain passes through LDS; that holds the left operands, which
// prep writes in the order in which the lanes read them (1 KB a fragment), and what
// the waves that make the outputs take from the chain's.
#include "gemv_device.h"
#include "host_state.h"
#include "launch_rules.h"
#include "mixer_device.h"

#include <type_traits>

using namespace mixer;

namespace {

constexpr int C = 64;                   // tokens of a chunk

struct GdnArgs {
    const void * q, * k, * v;
    void * out;
    const float * g, * beta, * state;
    float * state_out;
    const int32_t * slots, * starts;
    uint8_t * ws;
    int64_t q_tok, k_tok, v_tok, out_tok, gate_tok, n_states;
    int n_tok, n_seq, n_kh, n_vh, vd, tiled, chunks, out16;
    float scale, eps;
};

// bytes of the workspace: per chunk and key head the fragments of K, Q and K^T,
// per chunk and value head those of T and the masked QK^T and the row factors.
// Rows of 16-bit elements are one f16 term as they stand (but for the scaling, and
// what lies 2^32 below a row's largest, in bf16, which rounds at 2^-40 of it).
template <class T, int K>
struct Work {
    static constexpr int TERMS = sizeof(typename T::elem) == 4 ? 2 : 1;
    static constexpr int KF = C * K * 2 * TERMS;          // 4 m-tiles x K/32 steps x terms of 1 KB
    static constexpr int HEAD = 3 * KF;                   // K, Q, K^T
    static constexpr int TF = C * C * 3;                  // 6 of the 8 fragments: 32 x 32 above the diagonal are 0
    static constexpr int VEC = 2048;                      // c1, cq, t, a, w: 64 floats each, then e^Gc
    static constexpr int VHEAD = 2 * TF + VEC;
};
inline int64_t work_bytes(int64_t chunks, int n_kh, int n_vh, int k_dim, int elem) {
    const int64_t head = 3ll * C * k_dim * (elem == 4 ? 4 : 2), vhead = 2ll * C * C * 3 + 2048;
    return chunks * (n_kh * head + n_vh * vhead);
}

__device__ __forceinline__ int key_head(const GdnArgs & a, int hv) {
    return a.tiled ? hv % a.n_kh : hv / (a.n_vh / a.n_kh);
}
__device__ __forceinline__ float gate(float g) { return g < -1e4f ? -1e4f : g; }
// the state of a sequence, or -1
__device__ __forceinline__ int64_t slot_of(const GdnArgs & a, int seq) {
    const int64_t s = a.slots ? sload(a.slots, seq) : seq;
    return s >= 0 && s < a.n_states ? s : -1;
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// pow2(-e) takes x to 2^14 .. 2^15 (as far as both are normal numbers: from 2^-112 on); for 0, infinities and NaN as for 1
__device__ __forceinline__ int exponent(float x) {
    const int e = (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 255) - 127;
    return (e < -112 || e > 127 ? 0 : e) - 14;
}

// ------------------------------------------------------------ token by token
template <class T, int N>
__device__ __forceinline__ void load_n(const typename T::elem * p, float (&x)[N]) {
    constexpr int E = 16 / sizeof(typename T::elem);
#pragma unroll
    for (int i = 0; i < N; i += E) {
        float y[E];
        load_row<T>(p + i, y);
#pragma unroll
        for (int j = 0; j < E; ++j) x[i + j] = y[j];
    }
}

template <class T, int K>
__global__ void __launch_bounds__(128) gdn_step_kernel(GdnArgs a) {
    typedef typename T::elem elem;
    constexpr int N = K / 4;                              // rows of S of a lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = (a.vd + 31) / 32;
    const int hv = blockIdx.x / pairs % a.n_vh, seq = blockIdx.x / pairs / a.n_vh;
    const int col0 = 32 * (blockIdx.x % pairs) + 16 * wave;
    if (col0 >= a.vd) return;
    const int64_t slot = slot_of(a, seq);
    if (slot < 0) return;
    const int hk = key_head(a, hv), part = lane >> 4, col = col0 + (lane & 15);
    const int first = iclamp(sload(a.starts, seq), 0, a.n_tok), end = iclamp(sload(a.starts, seq + 1), 0, a.n_tok);
    const int64_t at = ((slot * a.n_vh + hv) * K + part * N) * a.vd + col;
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = a.state[at + (int64_t)j * a.vd];
    const elem * const q = reinterpret_cast<const elem *>(a.q) + (int64_t)hk * K + part * N;
    const elem * const k = reinterpret_cast<const elem *>(a.k) + (int64_t)hk * K + part * N;
    const elem * const v = reinterpret_cast<const elem *>(a.v) + (int64_t)hv * a.vd + col;
    elem * const out = reinterpret_cast<elem *>(a.out) + (int64_t)hv * a.vd + col;
    auto sum4 = [](float x) {                             // over the 4 parts
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    };
    for (int t = first; t < end; ++t) {
        float kk[N], qq[N];
        load_n<T>(k + (int64_t)t * a.k_tok, kk);
        load_n<T>(q + (int64_t)t * a.q_tok, qq);
        const float vt = T::to(v[(int64_t)t * a.v_tok]);
        const float decay = expf(gate(a.g[(int64_t)t * a.gate_tok + hv])), beta = a.beta[(int64_t)t * a.gate_tok + hv];
        float x = 0.0f, y = 0.0f, qk = 0.0f, k2 = 0.0f, q2 = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            x = fmaf(s[j], kk[j], x);
            y = fmaf(s[j], qq[j], y);
            qk = fmaf(qq[j], kk[j], qk);
            if (a.eps > 0.0f) {
                k2 = fmaf(kk[j], kk[j], k2);
                q2 = fmaf(qq[j], qq[j], q2);
            }
        }
        x = sum4(x);
        y = sum4(y);
        qk = sum4(qk);
        float fk = 1.0f, fq = a.scale;
        if (a.eps > 0.0f) {
            fk = 1.0f / sqrtf(sum4(k2) + a.eps);
            fq *= 1.0f / sqrtf(sum4(q2) + a.eps);
        }
        const float u = beta * (vt - decay * (x * fk));
        const float uk = u * fk;
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = fmaf(kk[j], uk, s[j] * decay);
        if (part == 0) out[(int64_t)t * a.out_tok] = T::from(fq * fmaf(qk, uk, decay * y));
    }
#pragma unroll
    for (int j = 0; j < N; ++j) a.state_out[at + (int64_t)j * a.vd] = s[j];
}

// ---------------------------------------------------------------------- chunks
// elements at .. at + N - 1 of the two f16 terms of x down (less than 2^15)
template <int N>
__device__ __forceinline__ void split(const float * x, float down, v8h & hi, v8h & lo, int at) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        uint32_t u = __builtin_bit_cast(uint32_t, v2h{(_Float16)(x[j] * down), (_Float16)(x[j + 1] * down)});
        asm("" : "+v"(u));                                // or each is converted a second time for its rest
        const v2h h = __builtin_bit_cast(v2h, u);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            hi[at + j + i] = h[i];
            lo[at + j + i] = (_Float16)fmaf(x[j + i], down, -(float)h[i]);
        }
    }
}

// the largest of the 4 lanes that hold a column
__device__ __forceinline__ float over_column(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    uint32_t a = p[0], b = p[1];
    asm("" : "+v"(a), "+v"(b));                           // they differ, though the operands do not
    const uint32_t m = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    const auto q = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    uint32_t c = q[0], d = q[1];
    asm("" : "+v"(c), "+v"(d));
    return fmaxf(__builtin_bit_cast(float, c), __builtin_bit_cast(float, d));
}

// A workgroup per chunk and key head: K K^T and Q K^T once, by 16 rows a wave, then
// T and the masked Q K^T of its value heads, a wave each for up to 4 at a time: a
// head alone on 4 waves is a chain of barriers and of a triangular solve that does
// not fill them.  The heads' C x C matrices take the place of K and Q in LDS, one
// after the other, so that two workgroups share a CU.  2048 tokens, 16 key and 48
// value heads of 128 (MI355X): 25 us fp32, of which the rows of K and Q take 4, the
// two squares 5, the inverse 4; 93 MB written.
template <class T, int K>
__global__ void __launch_bounds__(256) gdn_prep_kernel(GdnArgs a) {
    typedef typename T::elem elem;
    typedef Work<T, K> W;
    constexpr int TERMS = W::TERMS;
    constexpr int P = K + 8;                              // halves of a row: 16 rows of 16 bytes meet all banks
    constexpr int M = 68;                                 // floats of a row of the C x C matrices
    constexpr int SM = K / 32;
    constexpr int PL = 2 * TERMS * C * P * 2, LX = 4 * C * M * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[PL > LX ? PL : LX];
    _Float16 (* const pl)[C][P] = reinterpret_cast<_Float16 (*)[C][P]>(lds);      // K's terms, Q's terms
    float (* const mat)[C][M] = reinterpret_cast<float (*)[C][M]>(lds);           // one a value head
    __shared__ __attribute__((aligned(16))) float Gh[4][C], Gl[4][C], fk[C], fq[C], bt[4][C];    // log2(e) G as two floats
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % a.n_kh, chunk = blockIdx.x / a.n_kh, per = a.n_vh / a.n_kh;
    const Tile tl = find_tile<C>(a.starts, nullptr, a.n_seq, a.n_tok, 1, chunk);
    if (tl.seq < 0) return;
    const int t0 = tl.first + tl.index * C, nt = min(C, tl.count - tl.index * C);
    uint8_t * const wk = a.ws + ((int64_t)chunk * a.n_kh + hk) * W::HEAD;
    auto head_of = [&](int r) { return a.tiled ? hk + r * a.n_kh : hk * per + r; };
    // g and beta of this wave's value head (r0 + wave), a token a lane: before the stores, which they would wait for
    float gate1 = 0.0f, beta1 = 0.0f;
    auto gates = [&](int r0) __attribute__((always_inline)) {
        if (r0 + wave >= per || lane >= nt) return;
        gate1 = a.g[(int64_t)(t0 + lane) * a.gate_tok + head_of(r0 + wave)];
        beta1 = a.beta[(int64_t)(t0 + lane) * a.gate_tok + head_of(r0 + wave)];
    };
    gates(0);

    // rows of K and Q: 4 threads each
    {
        constexpr int N = K / 4;
        const int row = tid >> 2, part = tid & 3;
        float x[2][N];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const elem * const p = reinterpret_cast<const elem *>(m ? a.q : a.k);
            load_n<T>(p + (int64_t)(t0 + min(row, nt - 1)) * (m ? a.q_tok : a.k_tok) + (int64_t)hk * K + part * N, x[m]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float ss = 0.0f, big = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (row >= nt) x[m][j] = 0.0f;
                ss = fmaf(x[m][j], x[m][j], ss);
                big = fmaxf(big, fabsf(x[m][j]));
            }
            ss += __shfl_xor(ss, 1);
            ss += __shfl_xor(ss, 2);
            big = fmaxf(big, __shfl_xor(big, 1));
            big = fmaxf(big, __shfl_xor(big, 2));
            const int e = exponent(big);
            float f = pow2(e);
            if (a.eps > 0.0f) f *= 1.0f / sqrtf(ss + a.eps);
            if (part == 0) (m ? fq : fk)[row] = f;
            const float down = pow2(-e);
#pragma unroll
            for (int j = 0; j < N; j += 8) {
                v8h hi, lo;
                split<8>(&x[m][j], down, hi, lo, 0);
                *reinterpret_cast<v8h *>(&pl[TERMS * m][row][part * N + j]) = hi;
                if (TERMS == 2) *reinterpret_cast<v8h *>(&pl[TERMS * m + 1][row][part * N + j]) = lo;
            }
        }
    }
    __syncthreads();

    // rows 16 wave .. of K K^T and Q K^T (element: column 16 n + l16, row 16 wave + 4 g + r), without the rows' factors
    v4f kk[4], qk[4];
    {
        v8h ka[SM][TERMS], qa[SM][TERMS];
#pragma unroll
        for (int s = 0; s < SM; ++s)
#pragma unroll
            for (int k = 0; k < TERMS; ++k) {
                ka[s][k] = *reinterpret_cast<const v8h *>(&pl[k][16 * wave + l16][32 * s + 8 * g]);
                qa[s][k] = *reinterpret_cast<const v8h *>(&pl[TERMS + k][16 * wave + l16][32 * s + 8 * g]);
            }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            kk[n] = qk[n] = v4f{};
            if (n <= wave) {
#pragma unroll
                for (int s = 0; s < SM; ++s) {
                    const v8h bh = *reinterpret_cast<const v8h *>(&pl[0][16 * n + l16][32 * s + 8 * g]);
                    if constexpr (TERMS == 2) {
                        const v8h bl = *reinterpret_cast<const v8h *>(&pl[1][16 * n + l16][32 * s + 8 * g]);
                        kk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][1], bh, kk[n], 0, 0, 0);
                        qk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][1], bh, qk[n], 0, 0, 0);
                        kk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][0], bl, kk[n], 0, 0, 0);
                        qk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][0], bl, qk[n], 0, 0, 0);
                    }
                    kk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][0], bh, kk[n], 0, 0, 0);
                    qk[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][0], bh, qk[n], 0, 0, 0);
                }
            }
        }
    }
    // the fragments of K, Q (m-tile of 16 tokens, steps of 32 dims) and K^T (m-tile of 16 dims, steps of 32 tokens)
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    for (int f = wave; f < 4 * SM; f += 4) {
        const int mt = f / SM, ks = f % SM, row = 16 * mt + l16;
#pragma unroll
        for (int k = 0; k < 2 * TERMS; ++k) {
            const v4h x = *reinterpret_cast<const v4h *>(&pl[k][row][32 * ks + 4 * g]);
            const v4h y = *reinterpret_cast<const v4h *>(&pl[k][row][32 * ks + 16 + 4 * g]);
            *reinterpret_cast<v8h *>(wk + (k / TERMS) * W::KF + (TERMS * f + k % TERMS) * 1024 + 16 * lane) =
                __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    for (int f = wave; f < K / 8; f += 4) {
        const int mt = f >> 1, ks = f & 1, dim = 16 * mt + l16;
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
            v8h x;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = pl[k][32 * ks + (j < 4 ? 4 * g + j : 12 + 4 * g + j)][dim];
            *reinterpret_cast<v8h *>(wk + 2 * W::KF + (TERMS * f + k) * 1024 + 16 * lane) = x;
        }
    }

    // this wave's C x C matrix, its columns times col, as fragments (m-tile mt, step ks) and a factor of each row
    float (* const X)[M] = mat[wave];
    auto put_square = [&](const float * col, uint8_t * to, float * factor) __attribute__((always_inline)) {
        float c[2][8];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) c[ks][j] = col ? col[32 * ks + (j < 4 ? 4 * g + j : 12 + 4 * g + j)] : 1.0f;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            float x[2][8], big = 0.0f;
#pragma unroll
            for (int ks = 0; ks <= mt / 2; ++ks) {
                const v4f y = *reinterpret_cast<const v4f *>(&X[16 * mt + l16][32 * ks + 4 * g]);
                const v4f z = *reinterpret_cast<const v4f *>(&X[16 * mt + l16][32 * ks + 16 + 4 * g]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[ks][j] = (j < 4 ? y[j & 3] : z[j & 3]) * c[ks][j];
                    big = fmaxf(big, fabsf(x[ks][j]));
                }
            }
            const int e = exponent(over_column(big));
            if (g == 0) factor[16 * mt + l16] = pow2(e);
            const float down = pow2(-e);
#pragma unroll
            for (int ks = 0; ks <= mt / 2; ++ks) {
                v8h hi, lo;
                split<8>(x[ks], down, hi, lo, 0);
                const int f = ks ? mt + 2 : mt;
                *reinterpret_cast<v8h *>(to + (2 * f) * 1024 + 16 * lane) = hi;
                *reinterpret_cast<v8h *>(to + (2 * f + 1) * 1024 + 16 * lane) = lo;
            }
        }
    };
    auto in_wave = []() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };   // other lanes read it
#pragma unroll 1
    for (int r0 = 0; r0 < per; r0 += 4) {
        const int heads = min(4, per - r0);
        const bool mine = wave < heads;
        uint8_t * const wv = a.ws + (int64_t)a.chunks * a.n_kh * W::HEAD +
                             ((int64_t)chunk * a.n_vh + head_of(r0 + (mine ? wave : 0))) * W::VHEAD;
        float * const vec = reinterpret_cast<float *>(wv + 2 * W::TF);
        if (mine) {
            // the sums of g, in fp64
            double s = lane < nt ? (double)gate(gate1) * 1.4426950408889634 : 0.0;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(s, d);
                if (lane >= d) s += o;
            }
            const float h = (float)s;
            Gh[wave][lane] = h;
            Gl[wave][lane] = (float)(s - (double)h);
            bt[wave][lane] = lane < nt ? beta1 : 0.0f;
        }
        gates(r0 + 4);
        __syncthreads();                                  // (and: K and Q, or the last heads' matrices, have been read)

        // rows 16 wave .. of every head's matrices: Q K^T with its decay in LDS, L in registers until that has been read
        float L[4][4][4];
        const int row = 16 * wave + 4 * g;
        const v4f fqi = *reinterpret_cast<const v4f *>(&fq[row]), fki = *reinterpret_cast<const v4f *>(&fk[row]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < heads) {
                const v4f hi = *reinterpret_cast<const v4f *>(&Gh[r][row]), lo = *reinterpret_cast<const v4f *>(&Gl[r][row]);
                const v4f bi = *reinterpret_cast<const v4f *>(&bt[r][row]);
                int under = row - l16;
                asm("" : "+v"(under));                    // or 32 comparisons are kept for all heads, and spilled
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (n <= (wave | 1)) {                // (block n = wave + 1 of even waves: the zeros beside the diagonal)
                        const int j = 16 * n + l16;
                        const float hj = Gh[r][j], lj = Gl[r][j], fj = fk[j];
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) {
                            const float d = __builtin_amdgcn_exp2f((hi[i4] - hj) + (lo[i4] - lj)) * fj;
                            mat[r][row + i4][j] = 16 * n <= under + i4 ? qk[n][i4] * (a.scale * fqi[i4]) * d : 0.0f;
                            L[r][n][i4] = 16 * n < under + i4 ? kk[n][i4] * (bi[i4] * fki[i4]) * d : 0.0f;
                        }
                    }
            }
        __syncthreads();
        if (mine) put_square(nullptr, wv + W::TF, vec + 3 * C);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < heads)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (n <= (wave | 1))
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) mat[r][row + i4][16 * n + l16] = L[r][n][i4];
        __syncthreads();
        if (mine) {
            // X = (I + L)^-1 in L's place.  Diagonal blocks of 16 (block g: a lane per column): forward substitution
            {
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float s = l16 == i ? 1.0f : 0.0f;
#pragma unroll
                    for (int l = 0; l < i; ++l) s = fmaf(-X[16 * g + i][16 * g + l], x[l], s);
                    x[i] = s;
                }
                in_wave();
#pragma unroll
                for (int i = 0; i < 16; ++i) X[16 * g + i][16 * g + l16] = x[i];
                in_wave();
            }
            // below it, first for the two diagonal blocks of 32, then for the whole: with Y = L_21 X_11, X_21 = -X_22 Y
            auto mul = [&](int i, int l, int j, v4f & to) __attribute__((always_inline)) {    // blocks of 16: to += (i, l) (l, j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    to = __builtin_amdgcn_mfma_f32_16x16x4f32(X[16 * i + l16][16 * l + 4 * k + g], X[16 * l + 4 * k + g][16 * j + l16], to, 0, 0, 0);
            };
            auto put = [&](int i, int j, const v4f & x, float sign) __attribute__((always_inline)) {
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) X[16 * i + 4 * g + i4][16 * j + l16] = sign * x[i4];
            };
            {
                v4f x = {}, y = {};
                mul(1, 0, 0, x), mul(3, 2, 2, y);
                in_wave();
                put(1, 0, x, 1.0f), put(3, 2, y, 1.0f);
                in_wave();
                x = y = v4f{};
                mul(1, 1, 0, x), mul(3, 3, 2, y);
                in_wave();
                put(1, 0, x, -1.0f), put(3, 2, y, -1.0f);
                in_wave();
            }
            {
                v4f x[2][2] = {};
#pragma unroll
                for (int i = 0; i < 2; ++i) mul(2 + i, 0, 0, x[i][0]), mul(2 + i, 1, 1, x[i][1]);
#pragma unroll
                for (int i = 0; i < 2; ++i) mul(2 + i, 1, 0, x[i][0]);
                in_wave();
#pragma unroll
                for (int i = 0; i < 2; ++i) put(2 + i, 0, x[i][0], 1.0f), put(2 + i, 1, x[i][1], 1.0f);
                in_wave();
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) x[i][j] = v4f{}, mul(2 + i, 2 + i, j, x[i][j]);
#pragma unroll
                for (int j = 0; j < 2; ++j) mul(3, 2, j, x[1][j]);
                in_wave();
#pragma unroll
                for (int i = 0; i < 2; ++i) put(2 + i, 0, x[i][0], -1.0f), put(2 + i, 1, x[i][1], -1.0f);
                in_wave();
            }
            put_square(bt[wave], wv, vec + 2 * C);        // T
            // the other factors of the rows
            const float hi = Gh[wave][lane], lo = Gl[wave][lane];
            const float e = __builtin_amdgcn_exp2f(hi + lo);
            vec[lane] = e * fk[lane];
            vec[C + lane] = e * fq[lane] * a.scale;
            vec[4 * C + lane] = __builtin_amdgcn_exp2f((Gh[wave][C - 1] - hi) + (Gl[wave][C - 1] - lo)) * fk[lane];
            vec[5 * C + lane] = __builtin_amdgcn_exp2f(Gh[wave][C - 1] + Gl[wave][C - 1]);
        }
        if (r0 + 4 < per) __syncthreads();                // G, bt and the matrices are written anew
    }
}

template <int N>
__device__ __forceinline__ float largest(const v4f (&x)[N]) {
    float big[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) big[j & 1] = fmaxf(big[j & 1], fabsf(x[i][j]));
    return over_column(fmaxf(big[0], big[1]));
}

// 16 PAIRS columns of a value head, 16 for each pair of waves, of which one has
// the chain, the other the outputs and the loads:
//   first:  S as operands, K S    | loads, the last chunk's outputs leave
//   second: U                     | Q S
//   third:  S                     | QK^T U, the outputs
// S as operands and U go from the one to the other through LDS.  A chunk's 180
// products (16-bit rows: 132) of 16 columns are 2900 clocks of MFMA; what bounds it
// is the chain of dependent instructions around them (largest of a column, split,
// convert, rescale) and the LDS reads before them.  One wave that does it all takes
// 11000 clocks a chunk, the pair 6700, of which U is 2600.
//   K, Q and K^T of a chunk follow one another through two buffers, each asked for
// a phase ahead: with a third one PAIRS = 4 would not fit beside fp32's fragments,
// and PAIRS = 2 gained nothing by it (within 2 %).
//   2 pairs or 4 (half the fragments' bytes through LDS, two waves to a SIMD):
// gdn_wide, which has the times.  MI355X, 48 value heads of 128 x 128, fp32, both kernels:
// 2048 tokens of new inputs 134 us (116 to 126 where the caches hold them from the call
// before), 8 sequences of 2048 690, that is 1.6 TB/s of K, Q, V and outputs.
template <class T, int K, int PAIRS>
__global__ void __launch_bounds__(128 * PAIRS) gdn_scan_kernel(GdnArgs a) {
    typedef typename T::elem elem;
    typedef Work<T, K> W;
    typedef elem Unit __attribute__((ext_vector_type(16 / sizeof(elem))));
    constexpr int KS = K / 32, KT = K / 16, TERMS = W::TERMS;
    constexpr int EB = sizeof(elem), UNITS = EB, RPI = 64 / UNITS;    // 16-byte units of 16 columns; rows of a load
    // LDS: K, Q and K^T in two buffers in turn, T, QK^T, factors; then for each pair V, U (and outputs), S as operands and its scale
    constexpr int AT_T = 2 * W::KF, AT_A = AT_T + W::TF, AT_VEC = AT_A + W::TF;
    constexpr int AT_V = AT_VEC + W::VEC, V_PAIR = C * 16 * EB, AT_U = AT_V + PAIRS * V_PAIR, U_PAIR = C * 16 * 4;
    constexpr int AT_S = AT_U + PAIRS * U_PAIR, S_PAIR = 2 * KS * 1024 + 256;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[AT_S + PAIRS * S_PAIR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4, pair = wave % PAIRS;
    const bool chain = wave < PAIRS;
    // a key head's workgroups, which share fragments, on one XCD (workgroups go to the 8 in turn)
    const int groups = (a.vd + 16 * PAIRS - 1) / (16 * PAIRS), per = a.n_vh / a.n_kh;
    const int at_once = min(a.n_kh, 8);
    int hk = blockIdx.x % at_once, rest = blockIdx.x / at_once;
    const int group = rest % groups;
    rest /= groups;
    const int head = rest % per;
    rest /= per;
    const int times = (a.n_kh + at_once - 1) / at_once;
    int seq = rest / times;
    hk += at_once * (rest % times);
    if (hk >= a.n_kh) return;
    const int hv = a.tiled ? hk + head * a.n_kh : hk * per + head;
    const int col0 = 16 * (PAIRS * group + pair);
    // the first token and the number of tokens of a sequence; chunks before it
    int first, count, chunk0 = 0;
    auto tokens = [&](int q, int & b) __attribute__((always_inline)) {
        b = iclamp(a.starts[q], 0, a.n_tok);
        return max(iclamp(a.starts[q + 1], 0, a.n_tok) - b, 0);
    };
    if (a.n_seq <= 64) {
        // the one with the seq-th most chunks (found bit by bit), as a workgroup that starts behind others with many
        // chunks is what the rest wait for (1 sequence of 1500 tokens behind 5 of 180, both kernels, us: bf16 128 ->
        // 106, fp32 159 -> 135)
        int b = 0, n = 0;
        if (lane < a.n_seq) n = tokens(lane, b);
        const int own = (n + C - 1) / C;
        uint64_t left = ~0ull >> (64 - a.n_seq);          // those it can be
        for (int bit = a.n_seq > 1 ? 31 - __builtin_clz(max(a.chunks, 1)) : -1; bit >= 0; --bit) {
            const uint64_t more = __ballot(own >> bit & 1) & left;
            const int those = __builtin_popcountll(more);
            left = seq < those ? more : left & ~more;
            seq -= seq < those ? 0 : those;
        }
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(left >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)left, 0));
        seq = __builtin_ctzll(__ballot((left >> lane & 1) && before == seq));
        first = __builtin_amdgcn_readlane(b, seq);
        count = __builtin_amdgcn_readlane(n, seq);
        if (lane < seq) chunk0 = own;
    } else {
        for (int s = lane; s < seq; s += 64) {
            int b;
            chunk0 = min(chunk0 + (tokens(s, b) + C - 1) / C, 1 << 24);    // (more than there are, if starts overlap)
        }
        first = iclamp(sload(a.starts, seq), 0, a.n_tok);
        count = max(iclamp(sload(a.starts, seq + 1), 0, a.n_tok) - first, 0);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) chunk0 += __shfl_xor(chunk0, d);
    chunk0 = __builtin_amdgcn_readfirstlane(chunk0);
    const int64_t slot = slot_of(a, seq);
    if (slot < 0) return;
    const bool work = col0 < a.vd;                        // the others load
    const int col = work ? col0 + l16 : 0;
    int chunks = (count + C - 1) / C;
    chunks = iclamp(chunks, 0, max(a.chunks - chunk0, 0));   // starts that overlap: what prep made, no more

    // (waves of the outputs) a run of 1 KB pieces for each, 4 of them an address
    const int loader = wave - PAIRS;
    auto copy = [&](const uint8_t * src, uint8_t * dst, auto bytes) __attribute__((always_inline)) {
        constexpr int N = decltype(bytes)::value / 1024, OWN1 = N / PAIRS;
        const auto from = buffer_of(src, N * 1024);
#pragma unroll
        for (int i = 0; i < OWN1; i += 4) {
            const int at = (loader * OWN1 + i) * 1024;
            dma16_at<0>(from, dst + at, 16 * lane, at);
            if (i + 1 < OWN1) dma16_at<1024>(from, dst + at, 16 * lane, at);
            if (i + 2 < OWN1) dma16_at<2 * 1024>(from, dst + at, 16 * lane, at);
            if (i + 3 < OWN1) dma16_at<3 * 1024>(from, dst + at, 16 * lane, at);
        }
        if (N % PAIRS != 0 && loader < N % PAIRS) {
            const int at = (N / PAIRS * PAIRS + loader) * 1024;
            dma16(from, dst + at, 16 * lane, at);
        }
    };
    auto key_part = [&](int c) __attribute__((always_inline)) { return a.ws + ((int64_t)(chunk0 + c) * a.n_kh + hk) * W::HEAD; };
    auto value_part = [&](int c) __attribute__((always_inline)) {
        return a.ws + (int64_t)a.chunks * a.n_kh * W::HEAD + ((int64_t)(chunk0 + c) * a.n_vh + hv) * W::VHEAD;
    };
    const std::integral_constant<int, W::KF> kf_bytes;
    const std::integral_constant<int, W::TF> tf_bytes;
    // the loads are there, and what the waves read of LDS before has been read
    auto sync = [&]() __attribute__((always_inline)) {
        pq2::wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // Products, up to 4 sums side by side (an MFMA waits for the one before it in its own): left fragments, of one
    // or two terms of 1 KB, read a group ahead of their use
    struct Left {
        v8h h[4], l[4];
    };
    const std::integral_constant<int, TERMS> own_terms;   // of K and Q
    const std::integral_constant<int, 2> two;
    auto products = [&](auto count, auto terms, auto width, auto place, auto use) __attribute__((always_inline)) {
        constexpr int N = decltype(count)::value;
        Left f[2];
        auto read = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < width(i)) {
                    const uint8_t * const p = place(i, k) + 16 * lane;
                    f[i & 1].h[k] = *reinterpret_cast<const v8h *>(p);
                    if (decltype(terms)::value == 2) f[i & 1].l[k] = *reinterpret_cast<const v8h *>(p + 1024);
                }
        };
        read(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i + 1 < N) read(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            use(i, f[i & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto four = [](int) __attribute__((always_inline)) { return 4; };
    auto mul = [](auto terms, int n, const Left & f, const v8h & hi, const v8h & lo, v4f * const (&to)[4]) __attribute__((always_inline)) {
        if constexpr (decltype(terms)::value == 2)
#pragma unroll
            for (int k = 0; k < n; ++k) *to[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.l[k], hi, *to[k], 0, 0, 0);
#pragma unroll
        for (int k = 0; k < n; ++k) *to[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h[k], lo, *to[k], 0, 0, 0);
#pragma unroll
        for (int k = 0; k < n; ++k) *to[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h[k], hi, *to[k], 0, 0, 0);
    };
    // half of a right fragment (elements 4 k ..) from a result tile, its columns scaled
    auto to_right = [](const v4f & x, float down, v8h & hi, v8h & lo, int k) __attribute__((always_inline)) {
        const float y[4] = {x[0], x[1], x[2], x[3]};
        split<4>(y, down, hi, lo, 4 * k);
    };
    // a C x C matrix times a right operand: step 0 for all m-tiles, step 1 for the lower two
    v4f x[4];
    auto square = [&](const uint8_t * base, const v4f (&right)[4], float down) __attribute__((always_inline)) {
        v8h rh[2], rl[2];
        to_right(right[0], down, rh[0], rl[0], 0);
        to_right(right[1], down, rh[0], rl[0], 1);
#pragma unroll
        for (int m = 0; m < 4; ++m) x[m] = v4f{};
        products(std::integral_constant<int, 2>{}, two, [](int i) __attribute__((always_inline)) { return i ? 2 : 4; },
                 [&](int i, int k) __attribute__((always_inline)) { return base + 2 * (4 * i + k) * 1024; },
                 [&](int i, const Left & f) __attribute__((always_inline)) {
                     v4f * const to[4] = {&x[2 * i], &x[2 * i + 1], &x[2], &x[3]};
                     mul(two, i ? 2 : 4, f, rh[i], rl[i], to);
                     if (!i) {
                         to_right(right[2], down, rh[1], rl[1], 0);
                         to_right(right[3], down, rh[1], rl[1], 1);
                     }
                 });
    };

    // V comes, and the outputs leave, as [row][16 columns], row 4 j + g of 16 being token 4 g + j, so that the 4 tokens
    // that the lanes read a column at lie in different banks
    auto token = [](int row) { return (row & ~15) + 4 * (row & 3) + (row >> 2 & 3); };
    const int row0 = lane / UNITS, unit0 = lane % UNITS;
    auto stage_v = [&](int c, uint8_t * to) __attribute__((always_inline)) {
        const int nt = min(C, count - c * C);
        const auto from = buffer_of(reinterpret_cast<const uint8_t *>(a.v) +
                                    ((int64_t)(first + c * C) * a.v_tok + (int64_t)hv * a.vd + col0) * EB,
                                    (int)((nt - 1) * a.v_tok + 16) * EB);    // past the last token: zeros
#pragma unroll
        for (int i = 0; i < C / RPI; ++i)
            dma16(from, to + 1024 * i, token(RPI * i + row0) * (int)a.v_tok * EB + 16 * unit0, 0);
    };
    auto put = [&](const uint8_t * from, int c) __attribute__((always_inline)) {
        const int nt = min(C, count - c * C);
        uint8_t * const to = reinterpret_cast<uint8_t *>(a.out) +
                             ((int64_t)(first + c * C) * a.out_tok + (int64_t)hv * a.vd + col0) * EB;
#pragma unroll
        for (int i = 0; i < C / RPI; ++i) {
            const int t = token(RPI * i + row0);
            const v4u x = *reinterpret_cast<const v4u *>(from + 1024 * i + 16 * lane);
            if (t < nt) {
                if (a.out16) *reinterpret_cast<v4u *>(to + (int64_t)t * a.out_tok * EB + 16 * unit0) = x;
                else
#pragma unroll
                    for (int j = 0; j < 16 / EB; ++j)
                        reinterpret_cast<elem *>(to + (int64_t)t * a.out_tok * EB + 16 * unit0)[j] =
                            __builtin_bit_cast(Unit, x)[j];
            }
        }
    };

    const int64_t at = ((slot * a.n_vh + hv) * K + 4 * g) * a.vd + col;
    v4f S[KT];                                            // (chain)
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = work && chain ? a.state[at + (int64_t)(16 * i + j) * a.vd] : 0.0f;
    float big = chain ? largest(S) : 0.0f, fs = 1.0f, fw = 1.0f, keep = 1.0f;
    v4f ks[4], cq[4], ca[4];                              // K S or Q S; the outputs' factors
    v8h rh[2], rl[2];                                     // w U as right operand
    auto column = [&](uint8_t * base) __attribute__((always_inline)) { return reinterpret_cast<elem *>(base) + 16 * g + l16; };

    auto outputs = [&](const uint8_t * __restrict__ af, uint8_t * __restrict__ u) __attribute__((always_inline)) {
        v4f Um[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) Um[m] = *reinterpret_cast<const v4f *>(u + 1024 * m + 16 * lane);
        const int e = exponent(largest(Um));
        square(af, Um, pow2(-e));
        const float fu = pow2(e);
        elem * const own = column(u);                     // (U has been read)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                own[(16 * m + 4 * j) * 16] = T::from(fmaf(x[m][j] * fu, ca[m][j], ks[m][j] * fs * cq[m][j]));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // other lanes read it
    };
    auto phase1 = [&](const uint8_t * __restrict__ k, uint8_t * __restrict__ q, uint8_t * __restrict__ t, uint8_t * __restrict__ vec,
                      uint8_t * __restrict__ v, const uint8_t * __restrict__ u, uint8_t * __restrict__ sf, int c) __attribute__((always_inline)) {
        if (!chain) {
            copy(key_part(c) + W::KF, q, kf_bytes);
            copy(value_part(c), t, tf_bytes);
            copy(value_part(c) + 2 * W::TF, vec, std::integral_constant<int, W::VEC>{});
            if (work) stage_v(c, v);
            if (work && c > 0) put(u, c - 1);
            return;
        }
        if (!work) return;
        const int e = exponent(big);
        const float down = pow2(-e);
        fs = pow2(e);
        *reinterpret_cast<float *>(sf + 2 * KS * 1024 + 4 * lane) = fs;
        v8h sh[2], sl[2];
        auto give = [&](int s) __attribute__((always_inline)) {
            *reinterpret_cast<v8h *>(sf + 2 * s * 1024 + 16 * lane) = sh[s & 1];
            *reinterpret_cast<v8h *>(sf + (2 * s + 1) * 1024 + 16 * lane) = sl[s & 1];
        };
        to_right(S[0], down, sh[0], sl[0], 0);
        to_right(S[1], down, sh[0], sl[0], 1);
        give(0);
#pragma unroll
        for (int m = 0; m < 4; ++m) ks[m] = v4f{};
        products(std::integral_constant<int, KS>{}, own_terms, four,
                 [&](int i, int m) __attribute__((always_inline)) { return k + TERMS * (m * KS + i) * 1024; },
                 [&](int i, const Left & f) __attribute__((always_inline)) {
                     v4f * const to[4] = {&ks[0], &ks[1], &ks[2], &ks[3]};
                     mul(own_terms, 4, f, sh[i & 1], sl[i & 1], to);
                     if (i + 1 < KS) {                    // the next step's right operand, between the products
                         to_right(S[2 * i + 2], down, sh[(i + 1) & 1], sl[(i + 1) & 1], 0);
                         to_right(S[2 * i + 3], down, sh[(i + 1) & 1], sl[(i + 1) & 1], 1);
                         give(i + 1);
                     }
                 });
    };
    auto phase2 = [&](uint8_t * __restrict__ k, const uint8_t * __restrict__ q, const uint8_t * __restrict__ t,
                      const uint8_t * __restrict__ vec, uint8_t * __restrict__ v, uint8_t * __restrict__ af, uint8_t * __restrict__ u,
                      const uint8_t * __restrict__ sf, int c) __attribute__((always_inline)) {
        if (!chain) {
            copy(key_part(c) + 2 * W::KF, k, kf_bytes);
            copy(value_part(c) + W::TF, af, tf_bytes);
        }
        if (!work) return;
        auto factor = [&](int which, int m) {
            return *reinterpret_cast<const v4f *>(vec + 4 * (which * C + 16 * m + 4 * g));
        };
        if (!chain) {
            fs = *reinterpret_cast<const float *>(sf + 2 * KS * 1024 + 4 * lane);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                ks[m] = v4f{};
                cq[m] = factor(1, m);
                ca[m] = factor(3, m);
            }
            products(std::integral_constant<int, KS>{}, own_terms, four,
                     [&](int i, int m) __attribute__((always_inline)) { return q + TERMS * (m * KS + i) * 1024; },
                     [&](int i, const Left & f) __attribute__((always_inline)) {
                         const v8h sh = *reinterpret_cast<const v8h *>(sf + 2 * i * 1024 + 16 * lane);
                         const v8h sl = *reinterpret_cast<const v8h *>(sf + (2 * i + 1) * 1024 + 16 * lane);
                         v4f * const to[4] = {&ks[0], &ks[1], &ks[2], &ks[3]};
                         mul(own_terms, 4, f, sh, sl, to);
                     });
            return;
        }
        v4f R[4], Um[4];
        const elem * const own = column(v);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const v4f f = factor(0, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) R[m][j] = fmaf(-f[j], ks[m][j] * fs, T::to(own[(16 * m + 4 * j) * 16]));
        }
        int e = exponent(largest(R));
        const float fr = pow2(e);
        square(t, R, pow2(-e));
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const v4f f = factor(2, m), w = factor(4, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) Um[m][j] = x[m][j] * fr * f[j];
            *reinterpret_cast<v4f *>(u + 1024 * m + 16 * lane) = Um[m];
#pragma unroll
            for (int j = 0; j < 4; ++j) Um[m][j] *= w[j];
        }
        e = exponent(largest(Um));
        fw = pow2(e);
        keep = *reinterpret_cast<const float *>(vec + 4 * 5 * C);
#pragma unroll
        for (int m = 0; m < 4; ++m) to_right(Um[m], pow2(-e), rh[m / 2], rl[m / 2], m & 1);
    };
    auto phase3 = [&](const uint8_t * __restrict__ kt, uint8_t * __restrict__ k, const uint8_t * __restrict__ af,
                      uint8_t * __restrict__ u, int c) __attribute__((always_inline)) {
        if (!chain) {
            if (c + 1 < chunks) copy(key_part(c + 1), k, kf_bytes);
            if (work) outputs(af, u);
            return;
        }
        if (!work) return;
        float top[2] = {0.0f, 0.0f};
        v4f y[4];
        products(std::integral_constant<int, KT / 2>{}, own_terms, four,
                 [&](int i, int k) __attribute__((always_inline)) { return kt + TERMS * (2 * (4 * (i / 2) + k) + (i & 1)) * 1024; },
                 [&](int i, const Left & f) __attribute__((always_inline)) {
                     if (!(i & 1)) y[0] = y[1] = y[2] = y[3] = v4f{};
                     v4f * const to[4] = {&y[0], &y[1], &y[2], &y[3]};
                     mul(own_terms, 4, f, rh[i & 1], rl[i & 1], to);
                     if (i & 1)
#pragma unroll
                         for (int k = 0; k < 4; ++k)
#pragma unroll
                             for (int j = 0; j < 4; ++j) {
                                 const float st = fmaf(y[k][j], fw, keep * S[4 * (i / 2) + k][j]);
                                 S[4 * (i / 2) + k][j] = st;
                                 top[k & 1] = fmaxf(top[k & 1], fabsf(st));
                             }
                 });
        big = over_column(fmaxf(top[0], top[1]));
    };

    uint8_t * const v = lds + AT_V + pair * V_PAIR, * const u = lds + AT_U + pair * U_PAIR, * const sf = lds + AT_S + pair * S_PAIR;
    if (chunks > 0 && !chain) copy(key_part(0), lds, kf_bytes);
#pragma clang loop unroll(disable)
    for (int c = 0; c < chunks; ++c) {
        uint8_t * const one = lds + (c & 1) * W::KF, * const two = lds + (~c & 1) * W::KF;
        sync();                                           // K is in the one
        phase1(one, two, lds + AT_T, lds + AT_VEC, v, u, sf, c);
        sync();                                           // Q is in the two, T, V and S as operands are there
        phase2(one, two, lds + AT_T, lds + AT_VEC, v, lds + AT_A, u, sf, c);
        sync();                                           // K^T is in the one, QK^T and U are there
        phase3(one, two, lds + AT_A, u, c);
    }
    if (chunks > 0 && work && !chain) put(u, chunks - 1);
    if (!work || !chain) return;
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) a.state_out[at + (int64_t)(16 * i + j) * a.vd] = S[i][j];
}

template <class T, int K>
int launch(const GdnArgs & a, bool chunked, hipStream_t s) {
    if (!chunked) {
        const int64_t blocks = (int64_t)a.n_seq * a.n_vh * ((a.vd + 31) / 32);
        hipLaunchKernelGGL((gdn_step_kernel<T, K>), dim3((unsigned)blocks), dim3(128), 0, s, a);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL((gdn_prep_kernel<T, K>), dim3((unsigned)((int64_t)a.chunks * a.n_kh)), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    // (8 key heads at a time, those that there are not return)
    const int64_t heads = (int64_t)a.n_seq * (a.n_vh / a.n_kh) * (a.n_kh < 8 ? a.n_kh : (a.n_kh + 7) / 8 * 8);
    auto scan = [&](auto pairs) {
        constexpr int P = decltype(pairs)::value;
        hipLaunchKernelGGL((gdn_scan_kernel<T, K, P>), dim3((unsigned)(heads * ((a.vd + 16 * P - 1) / (16 * P)))),
                           dim3(128 * P), 0, s, a);
    };
    if (pq2::gdn_wide((int64_t)a.n_seq * a.n_vh, a.vd, pq2host::device_info().cus)) scan(std::integral_constant<int, 4>{});
    else scan(std::integral_constant<int, 2>{});
    return (int)hipGetLastError();
}
template <class T>
int launch_k(int k, const GdnArgs & a, bool chunked, hipStream_t s) {
    return k == 128 ? launch<T, 128>(a, chunked, s) : launch<T, 64>(a, chunked, s);
}

// 1: invalid, 0: nothing to do, -1: to be run
int check(const bonsai_p40_gdn_args * p) {
    if (!p) return 1;
    if (p->k_dim != 64 && p->k_dim != 128) return 1;
    if (p->v_dim < 16 || p->v_dim > 256 || p->v_dim % 16 != 0) return 1;
    if (p->n_k_head < 1 || p->n_v_head < 1 || p->n_v_head > 65536 || p->n_v_head % p->n_k_head != 0) return 1;
    if (!is_type(p->type) || p->n_states < 0 || p->n_tok < 0 || p->max_new < 0) return 1;
    const int64_t kr = (int64_t)p->n_k_head * p->k_dim, vr = (int64_t)p->n_v_head * p->v_dim;
    const int per16 = 16 / type_bytes(p->type);
    if (p->q_tok < kr || p->k_tok < kr || p->q_tok % per16 != 0 || p->k_tok % per16 != 0) return 1;
    if (p->v_tok < vr || p->v_tok % per16 != 0 || p->v_tok > (1 << 22) || p->out_tok < vr || p->gate_tok < p->n_v_head) return 1;
    if (!(p->scale > -INFINITY && p->scale < INFINITY) || !(p->l2_eps >= 0.0f && p->l2_eps < INFINITY)) return 1;
    if (p->n_seq <= 0) return 0;
    if (p->n_tok > 0x7fffffff || p->n_states > (1ll << 40)) return 1;
    // a grid has fewer than 2^32 threads: 128 per 32 columns, twice that in chunks, where key heads are rounded up to 8
    if (p->n_tok > (1ll << 27) / p->n_v_head || p->n_seq >= (1ll << 20) / p->n_v_head) return 1;
    return -1;
}
int64_t chunks_of(const bonsai_p40_gdn_args * p) { return p->n_tok / C + (p->n_seq < p->n_tok ? p->n_seq : p->n_tok); }
bool chunked(const bonsai_p40_gdn_args * p) {
    const int64_t most = p->max_new > 0 && p->max_new < p->n_tok ? p->max_new : p->n_tok;
    return pq2::gdn_chunked(most);
}

}  // namespace

extern "C" int64_t bonsai_p40_gdn_workspace_bytes(const bonsai_p40_gdn_args * p) {
    return check(p) == -1 && chunked(p) ? work_bytes(chunks_of(p), p->n_k_head, p->n_v_head, p->k_dim, type_bytes(p->type)) : 0;
}

extern "C" int bonsai_p40_gdn(const bonsai_p40_gdn_args * p, bonsai_stream stream) {
    const int rc = check(p);
    if (rc >= 0) return rc;
    if (pq2host::any_null(p->starts)) return 1;
    if (p->n_states > 0 && pq2host::any_null(p->state, p->state_out)) return 1;
    if (p->n_tok > 0 && pq2host::any_null(p->q, p->k, p->v, p->out, p->g, p->beta)) return 1;
    const int e = type_bytes(p->type), per16 = 16 / e;
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->out, e) || !aligned(p->g, 4) ||
        !aligned(p->beta, 4) || !aligned(p->state, 4) || !aligned(p->state_out, 4) || !aligned(p->starts, 4) ||
        !aligned(p->slots, 4) || !aligned(p->workspace, 16))
        return 1;
    const bool ch = p->workspace != nullptr && chunked(p);
    if (ch && p->workspace_bytes < work_bytes(chunks_of(p), p->n_k_head, p->n_v_head, p->k_dim, type_bytes(p->type))) return 1;
    GdnArgs a;
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.out = p->out;
    a.g = p->g;
    a.beta = p->beta;
    a.state = p->state;
    a.state_out = p->state_out;
    a.slots = p->slots;
    a.starts = p->starts;
    a.ws = reinterpret_cast<uint8_t *>(p->workspace);
    a.q_tok = p->q_tok;
    a.k_tok = p->k_tok;
    a.v_tok = p->v_tok;
    a.out_tok = p->out_tok;
    a.gate_tok = p->gate_tok;
    a.n_states = p->n_states;
    a.n_tok = (int)p->n_tok;
    a.n_seq = p->n_seq;
    a.n_kh = p->n_k_head;
    a.n_vh = p->n_v_head;
    a.vd = p->v_dim;
    a.tiled = p->tiled != 0;
    a.chunks = (int)chunks_of(p);
    a.out16 = aligned(p->out, 16) && p->out_tok % per16 == 0;    // rows of out that take 16 bytes at a time
    a.scale = p->scale;
    a.eps = p->l2_eps;
    const hipStream_t s = (hipStream_t)stream;
    if (p->type == BONSAI_P40_F32) return launch_k<F32>(p->k_dim, a, ch, s);
    if (p->type == BONSAI_P40_F16) return launch_k<F16>(p->k_dim, a, ch, s);
    return launch_k<BF16>(p->k_dim, a, ch, s);
}
