// The rules of csrc/launch_rules.h for the token mixers as C functions, for
// tests/test_mixer_rules.py.
#include "../../p40-kernel_amd/csrc/launch_rules.h"

extern "C" {
int rope_tile(int columns, int64_t n_tok) { return pq2::rope_tile(columns != 0, n_tok); }
void attn_plan(int64_t n_tok, int64_t n_seq, int64_t group, int64_t n_kv, int64_t dim, int64_t max_kv, int64_t rows, int64_t cus,
               int64_t * out) {
    const pq2::AttnPlan p = pq2::attn_plan(n_tok, n_seq, group, n_kv, dim, max_kv, rows, cus);
    out[0] = p.keys;
    out[1] = p.tiles;
    out[2] = p.chunk;
    out[3] = p.n_split;
}
int attn_join_wide(int64_t n_split) { return pq2::attn_join_wide(n_split); }
int gdn_chunked(int64_t max_new) { return pq2::gdn_chunked(max_new); }
int gdn_wide(int64_t heads, int64_t v_dim, int64_t cus) { return pq2::gdn_wide(heads, v_dim, cus); }
}
