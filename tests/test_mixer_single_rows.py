"""CPU: the stride of a dimension that has one entry says nothing, and is not what a
token mixer's wrapper refuses a call for."""
import pytest

import bonsai_p40 as B
from test_mixer_args import read

torch = pytest.importorskip("torch")
z, i32, f16 = torch.zeros, torch.int32, torch.float16


def one_row(heads, dim, dtype, wide=7):
    """The first token of several, whose heads are inside rows of a width that no 16-byte rows have."""
    return z(3, heads * dim + wide, dtype=dtype)[:, :heads * dim].view(3, heads, dim)[:1]


def attn(**change):
    kw = dict(q=z(1, 4, 64, dtype=f16), k_pages=z(3, 2, 16, 64, dtype=f16), v_pages=z(3, 2, 16, 64, dtype=f16),
              table=z(1, 3, dtype=i32), starts=z(2, dtype=i32), kv_len=z(1, dtype=i32), out=z(1, 4, 64, dtype=f16),
              workspace=None, max_kv=0, scale=None)
    return read(B.AttnPagedArgs, B._attn_args(**{**kw, **change}))


def test_one_token_inside_an_odd_row():
    a = attn(q=one_row(4, 64, f16), out=one_row(4, 64, f16))
    assert a.q_tok == a.out_tok == 256                     # a multiple of 8 elements, as two tokens' would have to be
    t = dict(q=z(1, 4, 64), k=z(1, 2, 64), v=z(1, 2, 64), q_norm=None, k_norm=None, eps=1e-6, pos=z(1, dtype=i32),
             inv_freq=None, slots=z(1, dtype=torch.int64), k_pages=z(3, 2, 16, 64, dtype=f16),
             v_pages=z(3, 2, 16, 64, dtype=f16), q_out=one_row(4, 64, f16), interleaved=False)
    assert read(B.QkNormRopeArgs, B._qk_norm_rope_args(**t)).q_out_tok == 256
    rows = [one_row(2, 64, torch.float32) for _ in range(2)] + [one_row(4, 32, torch.float32)]
    g = read(B.GdnArgs, B._gdn_args(*rows, z(1, 4), z(1, 4), z(1, 4, 64, 32), z(1, 4, 64, 32), one_row(4, 32, torch.float32),
                                    z(2, dtype=i32), None, 0, None, None, 0.0, False))
    assert (g.q_tok, g.k_tok, g.v_tok, g.out_tok) == (128, 128, 128, 128)


def test_two_tokens_inside_odd_rows_keep_their_stride():
    q = z(2, 4 * 64 + 7, dtype=f16)[:, :256].view(2, 4, 64)
    assert attn(q=q, out=z(2, 4, 64, dtype=f16), starts=z(2, dtype=i32)).q_tok == 263      # which the library refuses


def test_one_page_inside_odd_ones():
    wide = z(3, 2 * 16 * 64 + 5, dtype=f16)[:, :2 * 16 * 64].view(3, 2, 16, 64)[:1]
    assert attn(k_pages=wide, v_pages=wide).page_stride == 2048
    assert attn(k_pages=wide, v_pages=z(1, 2, 16, 64, dtype=f16)).page_stride == 2048
    # one head: its stride is the page's
    a = attn(q=z(1, 4, 64, dtype=f16), k_pages=z(3, 4, 16, 64, dtype=f16)[:, 1:2], v_pages=z(3, 4, 16, 64, dtype=f16)[:, :1])
    assert (a.page_stride, a.n_kv_head) == (4096, 1)


def test_pages_of_other_strides_are_refused():
    for v in (z(3, 4, 16, 64, dtype=f16)[:, :2], z(3, 2, 16, 128, dtype=f16)[..., :64], z(3, 2, 64, 16, dtype=f16).transpose(2, 3)):
        with pytest.raises(ValueError):
            attn(v_pages=v)
