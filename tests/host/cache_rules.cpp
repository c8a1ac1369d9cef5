// The rules of csrc/launch_rules.h for 8-bit pages and shared prefixes as C functions, for
// tests/test_cache_rules.py.
#include "../../p40-kernel_amd/csrc/launch_rules.h"

static void put(const pq2::AttnPlan & p, int64_t * out) {
    out[0] = p.keys;
    out[1] = p.tiles;
    out[2] = p.chunk;
    out[3] = p.n_split;
}
extern "C" {
void attn_plan(int64_t n_tok, int64_t n_seq, int64_t group, int64_t n_kv, int64_t dim, int64_t max_kv, int64_t rows, int64_t cus,
               int bytes, int whole, int64_t * out) {
    put(pq2::attn_plan(n_tok, n_seq, group, n_kv, dim, max_kv, rows, cus, bytes != 0, whole != 0), out);
}
void attn_own_plan(int64_t n_tok, int64_t n_seq, int64_t group, int64_t n_kv, int64_t dim, int64_t max_kv, int64_t rows, int64_t cus,
                   int bytes, int64_t * out) {
    put(pq2::attn_own_plan(n_tok, n_seq, group, n_kv, dim, max_kv, rows, cus, bytes != 0), out);
}
int attn_seen(int before, int kv, int tok) { return pq2::attn_seen(before, kv, tok); }
int attn_one_launch(int64_t first, int64_t own) { return pq2::attn_one_launch(first, own); }
int read_streams(int64_t bytes) { return pq2::read_streams(bytes); }
}
