"""CPU: the rules that place the work over 8-bit pages and shared prefixes
(csrc/launch_rules.h), compiled with g++, for a card of 256 CUs."""
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
    so = str(tmp_path_factory.mktemp("rules") / "cache_rules.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    os.path.join(ROOT, "tests", "host", "cache_rules.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


def plan(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows=128, q8=False, whole=False):
    out = (I64 * 4)()
    rules.attn_plan(*map(I64, (n_tok, n_seq, group, n_kv, dim, max_kv, rows, CUS)), int(q8), int(whole), out)
    return bool(out[0]), out[1], out[2], out[3]


def own(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows=128, q8=False):
    out = (I64 * 4)()
    rules.attn_own_plan(*map(I64, (n_tok, n_seq, group, n_kv, dim, max_kv, rows, CUS)), int(q8), out)
    return bool(out[0]), out[1], out[2], out[3]


def test_plans_cover_the_work(rules):
    """Every ragged set of sequences, or of groups, finds its row tiles, every key its part."""
    rng = random.Random(7)
    for _ in range(2000):
        n_seq, n_kv, group = rng.choice((1, 2, 7, 64, 500)), rng.choice((1, 2, 8)), rng.choice((1, 4, 6, 16))
        dim, rows, q8 = rng.choice((64, 128, 256)), rng.choice((64, 128)), rng.random() < 0.5
        new = [rng.choice((0, 1, 1, 5, 33, 700)) for _ in range(n_seq)]
        n_tok = max(sum(new), 1)
        max_kv = rng.choice((1, 31, 32, 500, 4000, 131071, (1 << 31) - 1))
        for keys, tiles, chunk, n_split in (plan(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows, q8, rng.random() < 0.5),
                                            own(rules, n_tok, n_seq, group, n_kv, dim, max_kv, rows, q8)):
            bm = 32 if keys else rows
            assert tiles >= sum(-(-n * group // bm) for n in new)
            assert chunk % 32 == 0 and chunk * n_split >= max_kv and (n_split == 1 or chunk * (n_split - 1) < max_kv)
            assert 1 <= n_split <= 2048


def test_16_bit_pages_keep_their_plan(rules):
    """The plan without a prefix is that of 16-bit pages but where heads of 256 split the keys."""
    for n_tok, n_seq, dim, kv in ((1, 1, 128, 4000), (32, 32, 64, 12000), (777, 1, 256, 16000), (300, 9, 128, 5000)):
        assert plan(rules, n_tok, n_seq, 6, 4, dim, kv, q8=True) == plan(rules, n_tok, n_seq, 6, 4, dim, kv)
    a, b = plan(rules, 32, 32, 6, 4, 256, 12000), plan(rules, 32, 32, 6, 4, 256, 12000, q8=True)
    assert a[0] and b[0] and b[3] == 2 * a[3]               # two workgroups to a CU


def test_one_group_has_no_tile_to_spare(rules):
    keys, tiles, chunk, n_split = plan(rules, 64, 1, 6, 4, 256, 16000, whole=True)
    assert not keys and tiles == 3 and CUS * 3 // 4 < 3 * 4 * n_split <= CUS
    assert plan(rules, 64, 1, 6, 4, 256, 16000)[1] == 4
    assert plan(rules, 64, 2, 6, 4, 256, 16000, whole=True)[1] == 5


# timed with the parts of attn_plan and with these
@pytest.mark.parametrize("n_tok,n_seq,group,n_kv,dim,keys,q8,parts", [
    (64, 64, 6, 4, 256, 515, False, 1), (32, 32, 6, 4, 256, 1515, True, 4), (250, 40, 4, 8, 128, 315, False, 1),
    (4, 4, 6, 4, 256, 35, False, 1)])
def test_own_keys(rules, n_tok, n_seq, group, n_kv, dim, keys, q8, parts):
    assert own(rules, n_tok, n_seq, group, n_kv, dim, keys, q8=q8)[::3] == (True, parts)


@pytest.mark.parametrize("bytes_,past", [(0, 0), (49 << 20, 0), (64 << 20, 0), ((64 << 20) + 1, 1), (98 << 20, 1), (1 << 40, 1)])
def test_rows_read_back(rules, bytes_, past):
    assert rules.read_streams(I64(bytes_)) == past


def test_the_cache_kernels_keep_to_registers():
    import kernel_resources as kr
    if not (os.path.exists(kr.LIB) and os.path.exists(os.path.join(kr.LLVM, "llvm-readelf"))):
        pytest.skip("needs the built library and ROCm's llvm-readelf")
    found = {}
    for r in kr.kernel_resources():
        found.setdefault(kr.family(r), []).append(r)
    for f in ("attn_q8_kernel", "attn_kernel", "attn_join_kernel", "kv_read_kernel", "qk_norm_rope_kernel"):
        assert f in found, f
        assert all(kr.is_hot_path(r) for r in found[f]), f
        assert not [r["name"] for r in found[f] if r["scratch"] or r["vgpr_spill"] or r["sgpr_spill"]], f


@pytest.mark.parametrize("n_tok,n_seq,group,n_kv,dim,keys,q8", [
    (131071, 131072, 1, 64, 64, 1224732915, False), (131071, 131072, 1, 64, 128, 742069199, True), (65535, 65536, 2, 64, 64, 542213998, True),
    (8388607, 8388608, 1, 1, 256, 170, True), (1 << 20, 1 << 20, 8, 1, 256, (1 << 31) - 65536, False)])
def test_grids_of_the_largest_batches(rules, n_tok, n_seq, group, n_kv, dim, keys, q8):
    """Workgroups of 256 threads, fewer than 2^32 of these a grid."""
    _, tiles, _, parts = own(rules, n_tok, n_seq, group, n_kv, dim, keys, q8=q8)
    _, tiles1, _, parts1 = plan(rules, n_tok, n_seq, group, n_kv, dim, keys, q8=q8, whole=True)
    first, second = tiles1 * parts1 * n_kv, tiles * parts * n_kv
    assert 0 < first < 1 << 24 and 0 < second < 1 << 24
    assert rules.attn_one_launch(I64(first), I64(second)) == (first + second < 1 << 24)
    assert rules.attn_one_launch(I64(1), I64((1 << 24) - 2)) and not rules.attn_one_launch(I64(1), I64((1 << 24) - 1))


def test_keys_a_token_sees(rules):
    """Own keys: token t of n sees those up to its own, none where there are fewer keys than tokens behind it; shared
    ones: every token all of them.  At lengths up to the longest there is, with the most tokens."""
    rng = random.Random(3)
    longest, most = (1 << 31) - 65536, (1 << 24) - 1
    for kv in (0, 1, 2, 31, 40, 4000, 70000, longest - most - 1, longest - 65535, longest - 1, longest):
        for n in (1, 2, 5, 33, 65535, 65536, 70000, most):
            for t in {0, 1, n // 2, n - 2, n - 1, rng.randrange(n)}:
                if 0 <= t < n:
                    assert rules.attn_seen(kv - n, kv, t) == max(kv - n + t + 1, 0), (kv, n, t)
                    assert rules.attn_seen(kv, kv, t) == kv, (kv, n, t)


def test_own_keys_in_parts_of_32_steps_at_most(rules):
    """Up to 64 parts, unless the batch fills the card many times over."""
    for n_seq in (1, 6, 64, 300, 1000):
        for dim, q8 in ((64, False), (128, True), (256, False), (256, True)):
            for keys in (515, 2048, 4096, 4097, 16015, 60000, 131071):
                _, tiles, chunk, parts = own(rules, n_seq, n_seq, 6, 4, dim, keys, q8=q8)
                assert chunk <= 32 * (64 if dim == 256 else 128) or parts >= 60, (n_seq, dim, keys, chunk, parts)


@pytest.mark.parametrize("n_tok,n_seq,group,n_kv", [((1 << 14) - 1, 1 << 19, 1024, 1), (16383, 1 << 23, 16, 64), (255, 1 << 21, 65536, 1), (1, 1 << 23, 1, 1),
                                                    ((1 << 23) - 1, 1 << 20, 1, 1)])
def test_grids_of_batches_with_more_rows_than_tokens(rules, n_tok, n_seq, group, n_kv):
    for dim in (64, 128, 256):
        for keys in (1, 4000, 1 << 20, (1 << 31) - 65536):
            for q8 in (False, True):
                _, tiles, _, parts = own(rules, n_tok, n_seq, group, n_kv, dim, keys, q8=q8)
                assert 0 < tiles * parts * n_kv < 1 << 24, (dim, keys, q8, tiles, parts)
