"""CPU: what the token mixers refuse before any launch (1), the empty calls (0), the
workspace sizes, and the checks of the Python wrappers."""
import ctypes as C

import pytest

import bonsai_p40 as B
from test_library import _gpu_visible

torch = pytest.importorskip("torch")
A = 4096          # a 16-byte aligned placeholder address, never dereferenced


def make(cls, base, **change):
    a = cls()
    for k, v in {**base, **change}.items():
        setattr(a, k, v)
    return a


ROPE = dict(q=A, k=A, v=A, q_tok=4 * 512, q_head=512, q_el=1, k_tok=256, k_head=256, k_el=1, v_tok=256, v_head=256,
            v_el=1, n_tok=3, n_head=4, n_kv_head=1, head_dim=256, n_rot=64, interleaved=0, eps=1e-6, q_norm=A, k_norm=A,
            pos=A, inv_freq=A, slots=A, q_out=A, q_out_tok=1024, q_type=B.BF16, kv_type=B.BF16, k_pages=A, v_pages=A,
            n_pages=7, page_stride=16 * 256, page_size=16)
ATTN = dict(q=A, out=A, q_tok=1024, out_tok=1024, n_tok=3, n_seq=2, n_head=8, n_kv_head=2, head_dim=128, io_type=B.BF16,
            kv_type=B.BF16, scale=0.1, k_pages=A, v_pages=A, n_pages=9, page_stride=2 * 16 * 128, page_size=16,
            max_pages=4, table=A, table_stride=4, starts=A, kv_len=A, max_kv=0, workspace=None, workspace_bytes=0)
GDN = dict(q=A, k=A, v=A, out=A, q_tok=256, k_tok=256, v_tok=512, out_tok=512, g=A, beta=A, gate_tok=4, state=A,
           state_out=A, n_states=2, slots=None, starts=A, n_tok=100, n_seq=2, n_k_head=2, n_v_head=4, k_dim=128, v_dim=128,
           type=B.F32, tiled=0, scale=0.1, l2_eps=1e-6, max_new=0, workspace=None, workspace_bytes=0)
INF, NAN = float("inf"), float("nan")

REFUSED = {
    "qk_norm_rope": (B.QkNormRopeArgs, ROPE, [
        dict(head_dim=96), dict(head_dim=0), dict(n_head=0), dict(n_kv_head=0), dict(n_head=16385), dict(n_rot=-8),
        dict(n_rot=264), dict(n_rot=12), dict(q_type=3), dict(q_type=-1), dict(kv_type=B.F32), dict(kv_type=7),
        dict(page_size=0), dict(page_size=24), dict(page_size=1 << 17), dict(n_pages=-1), dict(page_stride=4095),
        dict(page_stride=16 * 256 + 4), dict(q_out_tok=1023), dict(q_out_tok=1028), dict(n_tok=1 << 31),
        dict(q_tok=7, q_el=3), dict(k_tok=2, k_el=2), dict(v_tok=2, v_el=5), dict(q=A + 2), dict(q_out=A + 8),
        dict(k_pages=A + 8), dict(v_pages=A + 2), dict(pos=A + 2), dict(inv_freq=A + 4), dict(slots=A + 4),
        dict(q_norm=A + 1), dict(k_norm=A + 2)]),
    "attn_paged": (B.AttnPagedArgs, ATTN, [
        dict(head_dim=80), dict(n_head=7), dict(n_head=0), dict(n_kv_head=0), dict(n_head=65538), dict(kv_type=B.F32),
        dict(io_type=B.F16), dict(io_type=9), dict(page_size=8), dict(page_size=48), dict(page_size=1 << 17),
        dict(n_pages=-1), dict(n_pages=1 << 31), dict(page_stride=4095), dict(page_stride=4100), dict(q_tok=1023),
        dict(q_tok=1028), dict(out_tok=1000), dict(out_tok=1025), dict(scale=0.0), dict(scale=-1.0), dict(scale=INF),
        dict(scale=NAN), dict(max_pages=-1), dict(max_pages=5), dict(max_pages=1 << 27, table_stride=1 << 27),
        dict(max_kv=-1), dict(n_tok=1 << 28), dict(n_seq=1 << 26), dict(n_tok=1 << 21), dict(n_tok=1 << 20, n_seq=1 << 20), dict(q=A + 8), dict(out=A + 8), dict(k_pages=A + 8),
        dict(v_pages=A + 4), dict(workspace=A + 8, workspace_bytes=1 << 30), dict(table=A + 1), dict(starts=A + 2),
        dict(kv_len=A + 2), dict(workspace=A, workspace_bytes=16, max_pages=1 << 16, table_stride=1 << 16)]),
    "gdn": (B.GdnArgs, GDN, [
        dict(k_dim=96), dict(k_dim=256), dict(v_dim=0), dict(v_dim=24), dict(v_dim=272), dict(n_k_head=0), dict(n_v_head=0),
        dict(n_v_head=5), dict(n_v_head=65538), dict(type=3), dict(n_states=-1), dict(n_tok=-1), dict(max_new=-1),
        dict(q_tok=255), dict(k_tok=258), dict(v_tok=511), dict(out_tok=511), dict(gate_tok=3), dict(scale=INF),
        dict(scale=NAN), dict(l2_eps=-1.0), dict(l2_eps=NAN), dict(l2_eps=INF), dict(n_tok=1 << 26), dict(n_seq=1 << 26),
        dict(n_seq=1 << 18), dict(v_tok=514), dict(v_tok=(1 << 22) + 4),
        dict(q=A + 8), dict(k=A + 4), dict(v=A + 8), dict(out=A + 1), dict(g=A + 2), dict(beta=A + 1), dict(state=A + 2),
        dict(state_out=A + 3), dict(starts=A + 2), dict(slots=A + 1), dict(workspace=A + 4, workspace_bytes=1 << 30),
        dict(workspace=A, workspace_bytes=1000)]),
}
NEEDED = {"qk_norm_rope": "q k v pos inv_freq slots q_out k_pages v_pages", "attn_paged": "q out k_pages v_pages table starts kv_len",
          "gdn": "q k v out g beta state state_out starts"}
EMPTY = {"qk_norm_rope": [dict(n_tok=0), dict(n_tok=-3, q=None)], "attn_paged": [dict(n_tok=0), dict(n_seq=0, q=None)],
         "gdn": [dict(n_seq=0, state=None), dict(n_seq=-1)]}
no_gpu = pytest.mark.skipif(_gpu_visible(), reason="passes placeholder pointers: only where no GPU can run them")


def call(name, a):
    return getattr(B.lib(), "bonsai_p40_" + name)(C.byref(a), None)


@no_gpu
@pytest.mark.parametrize("name", REFUSED)
def test_refused(name):
    cls, base, bad = REFUSED[name]
    assert call(name, make(cls, base)) > 1              # gets as far as the launch, which has no device
    for change in bad:
        assert call(name, make(cls, base, **change)) == 1, change
    for p in NEEDED[name].split():
        assert call(name, make(cls, base, **{p: None})) == 1, p
    for change in EMPTY[name]:
        assert call(name, make(cls, base, **change)) == 0, change
    assert getattr(B.lib(), "bonsai_p40_" + name)(None, None) == 1


@no_gpu
def test_pointers_that_may_be_null():
    assert call("qk_norm_rope", make(B.QkNormRopeArgs, ROPE, q_norm=None, k_norm=None, n_rot=0, pos=None, inv_freq=None)) > 1
    assert call("attn_paged", make(B.AttnPagedArgs, ATTN, max_pages=0, table=None)) > 1
    assert call("attn_paged", make(B.AttnPagedArgs, ATTN, n_pages=0, k_pages=None, v_pages=None)) > 1
    assert call("gdn", make(B.GdnArgs, GDN, n_tok=0, q=None, k=None, v=None, out=None, g=None, beta=None)) > 1
    assert call("gdn", make(B.GdnArgs, GDN, n_states=0, state=None, state_out=None)) > 1


def test_workspace_bytes():
    L = B.lib()

    def attn(**change):
        return L.bonsai_p40_attn_paged_workspace_bytes(C.byref(make(B.AttnPagedArgs, ATTN, **change)))

    def gdn(**change):
        return L.bonsai_p40_gdn_workspace_bytes(C.byref(make(B.GdnArgs, GDN, **change)))
    # a part is head_dim + 2 floats of each row
    long = dict(max_pages=1 << 16, table_stride=1 << 16, n_tok=2)
    n = attn(**long)
    assert n > 0 and n % (2 * 8 * 130 * 4) == 0
    assert attn() == 0 and attn(**long, head_dim=96) == 0 and attn(**long, max_kv=64) == 0
    assert attn(**{**long, "n_tok": 0}) == 0
    # a chunk of 64 tokens: K, Q and K^T of a key head and two 64 x 64 matrices (6 of their 8 blocks of 16 x 32) of a
    # value head, each as two f16 terms, and 2 KB of factors; 16-bit rows are one term
    chunks = 100 // 64 + 2
    assert gdn() == chunks * (2 * 3 * 64 * 128 * 4 + 4 * (2 * 64 * 64 * 3 + 2048))
    assert gdn(type=B.BF16) == chunks * (2 * 3 * 64 * 128 * 2 + 4 * (2 * 64 * 64 * 3 + 2048))
    assert gdn(max_new=1) == 0 and gdn(n_tok=2) == 0 and gdn(v_dim=24) == 0


def test_structs_match_the_header(tmp_path):
    """The ctypes structs have the header's sizes and offsets."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"qk_norm_rope_args": B.QkNormRopeArgs, "attn_paged_args": B.AttnPagedArgs, "gdn_args": B.GdnArgs}
    lines = [f'printf("%zu {s} .\\n", sizeof(bonsai_p40_{s}));' for s in structs]
    lines += [f'printf("%zu {s} {f}\\n", offsetof(bonsai_p40_{s}, {f}));' for s, c in structs.items() for f, _ in c._fields_]
    src = tmp_path / "sizes.cpp"
    src.write_text('#include "bonsai_p40.h"\n#include <cstdio>\nint main() {\n' + "\n".join(lines) + "\n}\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(root, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        n, s, f = line.split()
        assert int(n) == (C.sizeof(structs[s]) if f == "." else getattr(structs[s], f).offset), line


def read(cls, packed):
    assert len(packed) == C.sizeof(cls)
    return cls.from_buffer_copy(packed)


def test_wrappers_want_device_tensors():
    t = _tensors()
    with pytest.raises(ValueError):
        B.qk_norm_rope(*[t[k] for k in ("q", "k", "v", "q_norm", "k_norm", "eps", "pos", "inv_freq", "slots", "k_pages",
                                        "v_pages", "q_out")])


def _tensors():
    z = torch.zeros
    return dict(q=z(5, 4, 64), k=z(5, 2, 64), v=z(5, 2, 64), q_norm=z(64), k_norm=z(64), eps=1e-6, pos=z(5, dtype=torch.int32),
                inv_freq=z(16, dtype=torch.float64), slots=z(5, dtype=torch.int64), k_pages=z(3, 2, 16, 64, dtype=torch.float16),
                v_pages=z(3, 2, 16, 64, dtype=torch.float16), q_out=z(5, 4, 64, dtype=torch.float16), interleaved=False)


def test_wrapper_checks_rope():
    z = torch.zeros
    ok = _tensors()
    a = read(B.QkNormRopeArgs, B._qk_norm_rope_args(**ok))
    assert (a.n_tok, a.n_head, a.n_kv_head, a.head_dim, a.n_rot, a.page_size, a.n_pages) == (5, 4, 2, 64, 32, 16, 3)
    assert (a.q_tok, a.q_head, a.q_el, a.q_out_tok, a.page_stride, a.q_type, a.kv_type) == (256, 64, 1, 256, 2048, B.F16, B.F16)
    cols = read(B.QkNormRopeArgs, B._qk_norm_rope_args(**{**ok, "q": z(4, 64, 5).permute(2, 0, 1)}))
    assert (cols.q_tok, cols.q_head, cols.q_el) == (1, 320, 5)
    for bad in (dict(q=z(5, 4, 64, dtype=torch.float16)), dict(k=z(5, 2, 32)), dict(v=z(4, 2, 64)), dict(q_norm=z(63)),
                dict(pos=z(5)), dict(pos=z(4, dtype=torch.int32)), dict(inv_freq=z(16)), dict(slots=z(5, dtype=torch.int32)),
                dict(v_pages=z(2, 2, 16, 64, dtype=torch.float16)), dict(v_pages=z(3, 2, 16, 64, dtype=torch.bfloat16)),
                dict(q_out=z(5, 4, 32, dtype=torch.float16)), dict(q_out=z(5, 64, 4, dtype=torch.float16).transpose(1, 2)),
                dict(slots=z(10, dtype=torch.int64)[::2]), dict(q_out=z(5, 4, 64, dtype=torch.float64)),
                dict(k_pages=z(3, 16, 2, 64, dtype=torch.float16).transpose(1, 2),
                     v_pages=z(3, 16, 2, 64, dtype=torch.float16).transpose(1, 2)), dict(q=z(5, 256))):
        with pytest.raises(ValueError):
            B._qk_norm_rope_args(**{**ok, **bad})


def test_wrapper_checks_attn():
    z, i32 = torch.zeros, torch.int32
    t = _tensors()
    ok = dict(q=t["q_out"], k_pages=t["k_pages"], v_pages=t["v_pages"], table=z(2, 3, dtype=i32), starts=z(3, dtype=i32),
              kv_len=z(2, dtype=i32), out=z(5, 4, 64, dtype=torch.float16), workspace=None, max_kv=0, scale=None)
    a = read(B.AttnPagedArgs, B._attn_args(**ok))
    assert (a.n_tok, a.n_seq, a.n_head, a.n_kv_head, a.head_dim, a.max_pages, a.table_stride, a.scale) == (5, 2, 4, 2, 64, 3, 3, 0.125)
    for bad in (dict(out=z(5, 4, 64)), dict(out=z(5, 4, 63, dtype=torch.float16)), dict(table=z(2, 3)), dict(starts=z(2, dtype=i32)),
                dict(kv_len=z(3, dtype=i32)), dict(kv_len=z(2, dtype=torch.int64)), dict(table=z(3, 2, dtype=i32).t()),
                dict(k_pages=z(3, 2, 16, 32, dtype=torch.float16), v_pages=z(3, 2, 16, 32, dtype=torch.float16)),
                dict(q=z(5, 4, 128, dtype=torch.float16)[:, :, ::2]), dict(table=z(6, dtype=i32))):
        with pytest.raises(ValueError):
            B._attn_args(**{**ok, **bad})


def test_wrapper_checks_gdn():
    z, i32 = torch.zeros, torch.int32
    ok = dict(q=z(5, 2, 64), k=z(5, 2, 64), v=z(5, 4, 32), g=z(5, 4), beta=z(5, 4), state=z(3, 4, 64, 32),
              state_out=z(3, 4, 64, 32), out=z(5, 4, 32), starts=z(4, dtype=i32), workspace=None, max_new=0, slots=None,
              scale=None, l2_eps=0.0, tiled=False)
    a = read(B.GdnArgs, B._gdn_args(**ok))
    assert (a.n_tok, a.n_seq, a.n_k_head, a.n_v_head, a.k_dim, a.v_dim, a.n_states, a.gate_tok) == (5, 3, 2, 4, 64, 32, 3, 4)
    for bad in (dict(k=z(5, 2, 32)), dict(k=z(5, 2, 64, dtype=torch.float16)), dict(v=z(4, 4, 32)), dict(g=z(5, 3)),
                dict(beta=z(4, 5).t()), dict(beta=z(5, 8)[:, :4]), dict(state=z(3, 4, 32, 64)), dict(state_out=z(2, 4, 64, 32)),
                dict(state_out=z(3, 4, 32, 64).transpose(2, 3)), dict(starts=z(4)), dict(slots=z(2, dtype=i32)),
                dict(slots=z(3, dtype=torch.int64)), dict(out=z(5, 4, 32, dtype=torch.bfloat16)), dict(q=z(5, 128)),
                dict(v=z(5, 4, 64)[:, :, ::2])):
        with pytest.raises(ValueError):
            B._gdn_args(**{**ok, **bad})
