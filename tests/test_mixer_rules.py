"""CPU: the rules that choose a token mixer's kernel and its split from sizes alone
(csrc/launch_rules.h), compiled with g++, on both sides of their lines for a card
of 256 CUs."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256
I64 = ctypes.c_int64


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rules") / "mixer_rules.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    os.path.join(ROOT, "tests", "host", "mixer_rules.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


def plan(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows=128):
    out = (I64 * 4)()
    rules.attn_plan(*map(I64, (n_tok, n_seq, group, n_kv, dim, max_kv, rows, CUS)), out)
    return bool(out[0]), out[1], out[2], out[3]


@pytest.mark.parametrize("columns,n_tok,tokens", [
    (0, 1, 4), (0, 64, 4), (0, 65, 16), (0, 1 << 30, 16), (1, 64, 4), (1, 65, 16), (1, 512, 16), (1, 513, 32)])
def test_rope_tile(rules, columns, n_tok, tokens):
    assert rules.rope_tile(columns, I64(n_tok)) == tokens


# sizes timed with the keys and with the rows split over the waves, and the faster one
@pytest.mark.parametrize("n_tok,n_seq,group,n_kv,dim,max_kv,keys", [
    (1, 1, 6, 4, 256, 4000, True), (4, 1, 6, 4, 256, 16000, True), (8, 1, 6, 4, 256, 16000, False),
    (128, 32, 6, 4, 256, 4000, True), (256, 32, 6, 4, 256, 4000, False), (128, 16, 4, 8, 128, 2000, True),
    (256, 16, 4, 8, 128, 2000, False), (2048, 1, 6, 4, 256, 2048, False)])
def test_attn_shape(rules, n_tok, n_seq, group, n_kv, dim, max_kv, keys):
    assert plan(rules, n_tok, n_seq, group, n_kv, dim, max_kv)[0] == keys


def test_attn_plan_covers_the_work(rules):
    """Every ragged set of sequences finds its row tiles, every key its part."""
    rng = random.Random(5)
    for _ in range(2000):
        n_seq, n_kv, group = rng.choice((1, 2, 7, 64, 500)), rng.choice((1, 2, 8)), rng.choice((1, 4, 6, 16))
        dim, rows = rng.choice((64, 128, 256)), rng.choice((64, 128))
        new = [rng.choice((0, 1, 1, 5, 33, 700)) for _ in range(n_seq)]
        n_tok = max(sum(new), 1)
        max_kv = rng.choice((1, 31, 32, 500, 4000, 131071, (1 << 31) - 1))
        keys, tiles, chunk, n_split = plan(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows)
        bm = 32 if keys else rows
        assert tiles >= sum(-(-n * group // bm) for n in new)
        assert chunk % 32 == 0 and chunk * n_split >= max_kv and (n_split == 1 or chunk * (n_split - 1) < max_kv)
        assert n_split <= 2048


def test_attn_split_fills_the_card(rules):
    """A long context of a few tokens is shared by about every CU."""
    for n_tok in (1, 4, 8, 16, 32, 64):
        _, tiles, _, n_split = plan(rules, n_tok, 1, 6, 4, 256, 60000)
        assert 3 * CUS // 4 <= tiles * n_split * 4 <= 2 * CUS, n_tok


@pytest.mark.parametrize("n_split,wide", [(2, 0), (8, 0), (9, 1), (2048, 1)])
def test_attn_join(rules, n_split, wide):
    assert rules.attn_join_wide(I64(n_split)) == wide


@pytest.mark.parametrize("max_new,chunked", [(1, 0), (12, 0), (13, 0), (14, 1), (16, 1), (1 << 30, 1)])
def test_gdn_form(rules, max_new, chunked):
    assert rules.gdn_chunked(I64(max_new)) == chunked


# value heads of all sequences: timed with 32 and with 64 columns a workgroup
@pytest.mark.parametrize("heads,v_dim,wide", [(48, 128, 0), (64, 128, 0), (65, 128, 1), (96, 128, 1), (384, 128, 1), (256, 16, 0)])
def test_gdn_columns(rules, heads, v_dim, wide):
    assert rules.gdn_wide(I64(heads), I64(v_dim), I64(CUS)) == wide
