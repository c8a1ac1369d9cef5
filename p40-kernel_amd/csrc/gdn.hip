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
// two f16 terms (22 bits; rows of the left, columns of the right operand scaled by
// powers of two so that f16's range does not matter) and the products hi hi,
// hi lo and lo hi run on v_mfma_f32_16x16x32_f16, 5 times the rate of fp32's own
// matrix instructions.  G is summed and subtracted in fp64: after a strong decay
// the differences of fp32 sums would have no digits left.
//   In the scan a wave has 16 columns of S, R and U to itself: a result tile
// (lane: column, 4 rows 4 g .. 4 g + 3) is the next product's right operand as it
// stands, if the left one lists its contraction as 4 g + j, 16 + 4 g + j (j < 4).
// So nothing of the chain passes through LDS; that holds the left operands, which
// prep writes in the order in which the lanes read them (1 KB a fragment).
#include "host_state.h"
#include "launch_rules.h"
#include "mixer_device.h"

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
    int n_tok, n_seq, n_kh, n_vh, vd, tiled, chunks;
    float scale, eps;
};

// bytes of the workspace: per chunk and key head the fragments of K, Q and K^T,
// per chunk and value head those of T and the masked QK^T and the row factors
template <int K>
struct Work {
    static constexpr int KF = C * K * 4;                  // 4 m-tiles x K/32 steps x 2 terms of 1 KB
    static constexpr int HEAD = 3 * KF;                   // K, Q, K^T
    static constexpr int TF = C * C * 4;
    static constexpr int VEC = 2048;                      // c1, cq, t, a, w: 64 floats each, then e^Gc
    static constexpr int VHEAD = 2 * TF + VEC;
};
inline int64_t work_bytes(int64_t chunks, int n_kh, int n_vh, int k_dim) {
    const int64_t head = 3ll * C * k_dim * 4, vhead = 2ll * C * C * 4 + 2048;
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
// the power of two that takes x to [1, 2), within what fp32 can invert; 0 for 0, infinities and NaN
__device__ __forceinline__ int exponent(float x) {
    const int e = (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 255) - 127;
    return e < -100 || e > 126 ? 0 : e > 100 ? 100 : e;
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
// x (about 1 at most) as two f16 terms
__device__ __forceinline__ void split(float x, _Float16 & hi, _Float16 & lo) {
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}

template <class T, int K>
__global__ void __launch_bounds__(256) gdn_prep_kernel(GdnArgs a) {
    typedef typename T::elem elem;
    typedef Work<K> W;
    constexpr int P = K + 8;                              // halves of a row: 16 rows of 16 bytes meet all banks
    constexpr int M = 68;                                 // floats of a row of the C x C matrices
    constexpr int SM = K / 32;
    __shared__ __attribute__((aligned(16))) _Float16 pl[4][C][P];     // K hi, lo, Q hi, lo
    __shared__ float L[C][M], X[C][M];
    __shared__ float tmp[4][16][17];
    __shared__ double G[C];
    __shared__ float fk[C], fq[C], bt[C], rt[C], ra[C];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int hv = blockIdx.x % a.n_vh, chunk = blockIdx.x / a.n_vh;
    const Tile tl = find_tile<C>(a.starts, a.n_seq, a.n_tok, 1, chunk);
    if (tl.seq < 0) return;
    const int hk = key_head(a, hv), t0 = tl.first + tl.index * C, nt = min(C, tl.count - tl.index * C);
    const bool lead = a.tiled ? hv < a.n_kh : hv % (a.n_vh / a.n_kh) == 0;   // writes the key head's fragments
    uint8_t * const wk = a.ws + ((int64_t)chunk * a.n_kh + hk) * W::HEAD;
    uint8_t * const wv = a.ws + (int64_t)a.chunks * a.n_kh * W::HEAD + ((int64_t)chunk * a.n_vh + hv) * W::VHEAD;

    // rows of K and Q: 4 threads each
    {
        constexpr int N = K / 4;
        const int row = tid >> 2, part = tid & 3;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float x[N] = {};
            const elem * const p = reinterpret_cast<const elem *>(m ? a.q : a.k);
            if (row < nt) load_n<T>(p + (int64_t)(t0 + row) * (m ? a.q_tok : a.k_tok) + (int64_t)hk * K + part * N, x);
            float ss = 0.0f, big = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ss = fmaf(x[j], x[j], ss);
                big = fmaxf(big, fabsf(x[j]));
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
            for (int j = 0; j < N; ++j) split(x[j] * down, pl[2 * m][row][part * N + j], pl[2 * m + 1][row][part * N + j]);
        }
    }
    if (wave == 0) {
        const float gt = lane < nt ? gate(a.g[(int64_t)(t0 + lane) * a.gate_tok + hv]) : 0.0f;
        double s = (double)gt;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        G[lane] = s;
        bt[lane] = lane < nt ? a.beta[(int64_t)(t0 + lane) * a.gate_tok + hv] : 0.0f;
    }
    __syncthreads();

    // rows 16 wave .. of K K^T and Q K^T, in fp32; then L, and Q K^T with its decay in X
    {
        v8h ka[SM][2], qa[SM][2];
#pragma unroll
        for (int s = 0; s < SM; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                ka[s][k] = *reinterpret_cast<const v8h *>(&pl[k][16 * wave + l16][32 * s + 8 * g]);
                qa[s][k] = *reinterpret_cast<const v8h *>(&pl[2 + k][16 * wave + l16][32 * s + 8 * g]);
            }
        float top[4] = {};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            v4f kk = {}, qk = {};
            if (n <= wave) {
#pragma unroll
                for (int s = 0; s < SM; ++s) {
                    const v8h bh = *reinterpret_cast<const v8h *>(&pl[0][16 * n + l16][32 * s + 8 * g]);
                    const v8h bl = *reinterpret_cast<const v8h *>(&pl[1][16 * n + l16][32 * s + 8 * g]);
                    kk = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][1], bh, kk, 0, 0, 0);
                    kk = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][0], bl, kk, 0, 0, 0);
                    kk = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[s][0], bh, kk, 0, 0, 0);
                    qk = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][1], bh, qk, 0, 0, 0);
                    qk = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][0], bl, qk, 0, 0, 0);
                    qk = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[s][0], bh, qk, 0, 0, 0);
                }
            }
            const int j = 16 * n + l16;
            const double Gj = G[j];
            const float fj = fk[j];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * g + r;
                const float d = j <= i ? expf((float)(G[i] - Gj)) : 0.0f;
                L[i][j] = j < i ? bt[i] * (kk[r] * fk[i] * fj) * d : 0.0f;
                const float x = j <= i ? a.scale * (qk[r] * fq[i] * fj) * d : 0.0f;
                X[i][j] = x;
                top[r] = fmaxf(top[r], fabsf(x));
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top[r] = fmaxf(top[r], __shfl_xor(top[r], d));
            if (l16 == 0) ra[16 * wave + 4 * g + r] = pow2(exponent(top[r]));
        }
    }
    __syncthreads();

    // a fragment of a C x C matrix in LDS: m-tile mt, step ks, as two terms
    auto put_square = [&](const float (*m)[M], const float * scale, uint8_t * to) {
        for (int f = wave; f < 8; f += 4) {
            const int mt = f >> 1, ks = f & 1, row = 16 * mt + l16;
            const float down = 1.0f / scale[row];
            v8h hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 h, l;
                split(m[row][32 * ks + (j < 4 ? 4 * g + j : 12 + 4 * g + j)] * down, h, l);
                hi[j] = h;
                lo[j] = l;
            }
            *reinterpret_cast<v8h *>(to + (2 * f) * 1024 + 16 * lane) = hi;
            *reinterpret_cast<v8h *>(to + (2 * f + 1) * 1024 + 16 * lane) = lo;
        }
    };
    put_square(X, ra, wv + W::TF);
    if (lead) {
        // K, Q: m-tile of 16 tokens, steps of 32 dims; K^T: m-tile of 16 dims, steps of 32 tokens
        for (int f = wave; f < 4 * SM; f += 4) {
            const int mt = f / SM, ks = f % SM, row = 16 * mt + l16;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v8h x;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = pl[k][row][32 * ks + (j < 4 ? 4 * g + j : 12 + 4 * g + j)];
                *reinterpret_cast<v8h *>(wk + (k >> 1) * W::KF + (2 * f + (k & 1)) * 1024 + 16 * lane) = x;
            }
        }
        for (int f = wave; f < K / 8; f += 4) {
            const int mt = f >> 1, ks = f & 1, dim = 16 * mt + l16;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v8h x;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = pl[k][32 * ks + (j < 4 ? 4 * g + j : 12 + 4 * g + j)][dim];
                *reinterpret_cast<v8h *>(wk + 2 * W::KF + (2 * f + k) * 1024 + 16 * lane) = x;
            }
        }
    }
    __syncthreads();                                      // X is free

    // X = (I + L)^-1.  Diagonal blocks of 16: a lane per column, forward substitution
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = l16 == i ? 1.0f : 0.0f;
#pragma unroll
            for (int l = 0; l < i; ++l) s = fmaf(-L[16 * wave + i][16 * wave + l], x[l], s);
            x[i] = s;
        }
        if (g == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) X[16 * wave + i][16 * wave + l16] = x[i];
        // what is above the diagonal
        for (int n = wave + 1; n < 4; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) X[16 * wave + 4 * g + r][16 * n + l16] = 0.0f;
    }
    __syncthreads();
    // below it, wave j has block column j: X_ij = -X_ii sum_l L_il X_lj
    for (int i = wave + 1; i < 4; ++i) {
        v4f s = {};
        for (int l = wave; l < i; ++l)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(L[16 * i + l16][16 * l + 4 * k + g],
                                                         X[16 * l + 4 * k + g][16 * wave + l16], s, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) tmp[wave][4 * g + r][l16] = s[r];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // other lanes read it
        v4f x = {};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(X[16 * i + l16][16 * i + 4 * k + g], tmp[wave][4 * k + g][l16], x, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) X[16 * i + 4 * g + r][16 * wave + l16] = -x[r];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // other lanes read it
    }
    __syncthreads();
    // T = X diag(beta), and the largest element of its rows
    {
        const int row = tid >> 2, part = tid & 3;
        float big = 0.0f;
        for (int j = part; j < C; j += 4) {
            const float x = X[row][j] * bt[j];
            X[row][j] = x;
            big = fmaxf(big, fabsf(x));
        }
        big = fmaxf(big, __shfl_xor(big, 1));
        big = fmaxf(big, __shfl_xor(big, 2));
        if (part == 0) rt[row] = pow2(exponent(big));
    }
    __syncthreads();
    put_square(X, rt, wv);
    // factors of the rows
    if (tid < C) {
        float * const vec = reinterpret_cast<float *>(wv + 2 * W::TF);
        const float e = expf((float)G[tid]);
        vec[tid] = e * fk[tid];
        vec[C + tid] = e * fq[tid] * a.scale;
        vec[2 * C + tid] = rt[tid];
        vec[3 * C + tid] = ra[tid];
        vec[4 * C + tid] = expf((float)(G[C - 1] - G[tid])) * fk[tid];
        vec[5 * C + tid] = expf((float)G[C - 1]);
    }
}

// right operand from result tiles: columns scaled to about 1; the factor that
// takes a product back
template <int N>
__device__ __forceinline__ float to_right(const v4f (&x)[N], v8h (&hi)[N / 2], v8h (&lo)[N / 2]) {
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(x[i][j]));
    big = fmaxf(big, __shfl_xor(big, 16));
    big = fmaxf(big, __shfl_xor(big, 32));
    const int e = exponent(big);
    const float down = pow2(-e);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            _Float16 h, l;
            split(x[i][j] * down, h, l);
            hi[i / 2][4 * (i & 1) + j] = h;
            lo[i / 2][4 * (i & 1) + j] = l;
        }
    return pow2(e);
}

template <class T, int K>
__global__ void __launch_bounds__(256) gdn_scan_kernel(GdnArgs a) {
    typedef typename T::elem elem;
    typedef Work<K> W;
    constexpr int KS = K / 32, KT = K / 16;
    constexpr int REG1 = 2 * W::KF, REG2 = W::KF + W::VHEAD;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[REG1 + REG2];
    uint8_t * const r1 = lds, * const r2 = lds + REG1;    // K, Q | K^T, T, QK^T, factors
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int quads = (a.vd + 63) / 64;
    const int hv = blockIdx.x / quads % a.n_vh, seq = blockIdx.x / quads / a.n_vh;
    const int col0 = 64 * (blockIdx.x % quads) + 16 * wave;
    const int64_t slot = slot_of(a, seq);
    if (slot < 0) return;
    const bool work = col0 < a.vd;                        // the others stage
    const int col = work ? col0 + l16 : 0, hk = key_head(a, hv);
    const int first = iclamp(sload(a.starts, seq), 0, a.n_tok);
    const int count = max(iclamp(sload(a.starts, seq + 1), 0, a.n_tok) - first, 0);
    int chunks = (count + C - 1) / C;
    // the number of the first chunk: those of the sequences before
    int chunk0 = 0;
    for (int s = lane; s < seq; s += 64)
        chunk0 += (max(iclamp(a.starts[s + 1], 0, a.n_tok) - iclamp(a.starts[s], 0, a.n_tok), 0) + C - 1) / C;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) chunk0 += __shfl_xor(chunk0, d);
    chunk0 = __builtin_amdgcn_readfirstlane(chunk0);
    chunks = iclamp(chunks, 0, max(a.chunks - chunk0, 0));   // starts that overlap: what prep made, no more

    auto copy = [&](const uint8_t * src, uint8_t * dst, int bytes) __attribute__((always_inline)) {
        const auto from = buffer_of(src, bytes);
        for (int i = wave * 1024; i < bytes; i += 4096) dma16(from, dst + i, 16 * lane, i);
    };
    auto stage1 = [&](int c) __attribute__((always_inline)) {
        copy(a.ws + ((int64_t)(chunk0 + c) * a.n_kh + hk) * W::HEAD, r1, REG1);
    };
    auto stage2 = [&](int c) __attribute__((always_inline)) {
        copy(a.ws + ((int64_t)(chunk0 + c) * a.n_kh + hk) * W::HEAD + REG1, r2, W::KF);
        copy(a.ws + (int64_t)a.chunks * a.n_kh * W::HEAD + ((int64_t)(chunk0 + c) * a.n_vh + hv) * W::VHEAD,
             r2 + W::KF, W::VHEAD);
    };
    auto sync = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const int64_t at = ((slot * a.n_vh + hv) * K + 4 * g) * a.vd + col;
    v4f S[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = work ? a.state[at + (int64_t)(16 * i + j) * a.vd] : 0.0f;
    const elem * const v = reinterpret_cast<const elem *>(a.v) + (int64_t)hv * a.vd + col;
    elem * const out = reinterpret_cast<elem *>(a.out) + (int64_t)hv * a.vd + col;

    // acc[m] += left fragments (two terms, 1 KB each, [m][s]) . right
    auto product = [&](const uint8_t * left, int m, int s, int steps, const v8h & hi, const v8h & lo, v4f c) __attribute__((always_inline)) {
        const v8h ah = *reinterpret_cast<const v8h *>(left + (2 * (m * steps + s)) * 1024 + 16 * lane);
        const v8h al = *reinterpret_cast<const v8h *>(left + (2 * (m * steps + s) + 1) * 1024 + 16 * lane);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, hi, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, lo, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, hi, c, 0, 0, 0);
    };

    if (chunks > 0) stage1(0);
#pragma clang loop unroll(disable)
    for (int c = 0; c < chunks; ++c) {
        const int t0 = first + c * C, nt = min(C, count - c * C);
        sync();                                           // K, Q are there; r2 is free
        stage2(c);
        float vt[4][4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 16 * m + 4 * g + j;
                vt[m][j] = work && t < nt ? T::to(v[(int64_t)(t0 + t) * a.v_tok]) : 0.0f;
            }
        v8h sh[KS], sl[KS];
        const float fs = to_right(S, sh, sl);
        v4f ks[4], qs[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            ks[m] = v4f{};
            qs[m] = v4f{};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                ks[m] = product(r1, m, s, KS, sh[s], sl[s], ks[m]);
                qs[m] = product(r1 + W::KF, m, s, KS, sh[s], sl[s], qs[m]);
            }
        }
        sync();                                           // the rest is there; r1 is free
        if (c + 1 < chunks) stage1(c + 1);
        const uint8_t * const tf = r2 + W::KF, * const af = tf + W::TF;
        const float * const vec = reinterpret_cast<const float *>(af + W::TF);
        auto factor = [&](int which, int m) { return *reinterpret_cast<const v4f *>(vec + which * C + 16 * m + 4 * g); };
        v4f R[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const v4f f = factor(0, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) R[m][j] = fmaf(-f[j] * fs, ks[m][j], vt[m][j]);
        }
        v8h rh[2], rl[2];
        const float fr = to_right(R, rh, rl);
        v4f Um[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            v4f x = {};
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) x = product(tf, m, s, 2, rh[s], rl[s], x);
            const v4f f = factor(2, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) Um[m][j] = x[j] * f[j] * fr;
        }
        const float fu = to_right(Um, rh, rl);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            v4f x = {};
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) x = product(af, m, s, 2, rh[s], rl[s], x);
            const v4f f = factor(3, m), h = factor(1, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 16 * m + 4 * g + j;
                const float o = fmaf(x[j], f[j] * fu, h[j] * fs * qs[m][j]);
                if (work && t < nt) out[(int64_t)(t0 + t) * a.out_tok] = T::from(o);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const v4f f = factor(4, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) Um[m][j] *= f[j];
        }
        const float fw = to_right(Um, rh, rl), keep = vec[5 * C];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            v4f x = {};
#pragma unroll
            for (int s = 0; s < 2; ++s) x = product(r2, i, s, 2, rh[s], rl[s], x);
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = fmaf(x[j], fw, keep * S[i][j]);
        }
    }
    if (!work) return;
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
    hipLaunchKernelGGL((gdn_prep_kernel<T, K>), dim3((unsigned)((int64_t)a.chunks * a.n_vh)), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    const int64_t blocks = (int64_t)a.n_seq * a.n_vh * ((a.vd + 63) / 64);
    hipLaunchKernelGGL((gdn_scan_kernel<T, K>), dim3((unsigned)blocks), dim3(256), 0, s, a);
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
    if (p->v_tok < vr || p->out_tok < vr || p->gate_tok < p->n_v_head) return 1;
    if (!(p->scale > -INFINITY && p->scale < INFINITY) || !(p->l2_eps >= 0.0f && p->l2_eps < INFINITY)) return 1;
    if (p->n_seq <= 0) return 0;
    if (p->n_tok > 0x7fffffff || p->n_states > (1ll << 40)) return 1;
    if (p->n_tok + p->n_seq > (1ll << 27) / p->n_v_head) return 1;      // workgroups
    return -1;
}
int64_t chunks_of(const bonsai_p40_gdn_args * p) { return p->n_tok / C + (p->n_seq < p->n_tok ? p->n_seq : p->n_tok); }
bool chunked(const bonsai_p40_gdn_args * p) {
    const int64_t most = p->max_new > 0 && p->max_new < p->n_tok ? p->max_new : p->n_tok;
    return pq2::gdn_chunked(most, p->n_seq);
}

}  // namespace

extern "C" int64_t bonsai_p40_gdn_workspace_bytes(const bonsai_p40_gdn_args * p) {
    return check(p) == -1 && chunked(p) ? work_bytes(chunks_of(p), p->n_k_head, p->n_v_head, p->k_dim) : 0;
}

extern "C" int bonsai_p40_gdn(const bonsai_p40_gdn_args * p, bonsai_stream stream) {
    const int rc = check(p);
    if (rc >= 0) return rc;
    if (pq2host::any_null(p->starts)) return 1;
    if (p->n_states > 0 && pq2host::any_null(p->state, p->state_out)) return 1;
    if (p->n_tok > 0 && pq2host::any_null(p->q, p->k, p->v, p->out, p->g, p->beta)) return 1;
    const int e = type_bytes(p->type);
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, e) || !aligned(p->out, e) || !aligned(p->g, 4) ||
        !aligned(p->beta, 4) || !aligned(p->state, 4) || !aligned(p->state_out, 4) || !aligned(p->starts, 4) ||
        !aligned(p->slots, 4) || !aligned(p->workspace, 16))
        return 1;
    const bool ch = p->workspace != nullptr && chunked(p);
    if (ch && p->workspace_bytes < work_bytes(chunks_of(p), p->n_k_head, p->n_v_head, p->k_dim)) return 1;
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
    a.scale = p->scale;
    a.eps = p->l2_eps;
    const hipStream_t s = (hipStream_t)stream;
    if (p->type == BONSAI_P40_F32) return launch_k<F32>(p->k_dim, a, ch, s);
    if (p->type == BONSAI_P40_F16) return launch_k<F16>(p->k_dim, a, ch, s);
    return launch_k<BF16>(p->k_dim, a, ch, s);
}
