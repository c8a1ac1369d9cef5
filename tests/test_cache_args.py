"""CPU: what the calls on 8-bit pages and shared prefixes refuse before any launch
(1), the empty calls (0), the workspace sizes, and the checks of the Python wrappers."""
import ctypes as C
import os
import subprocess

import pytest

import bonsai_p40 as B
from test_mixer_args import A, ATTN, INF, NAN, ROPE, make, no_gpu, read

torch = pytest.importorskip("torch")
z, i8, i32, i64, f16 = torch.zeros, torch.int8, torch.int32, torch.int64, torch.float16

Q8_ROPE = {**ROPE, "kv_type": B.Q8, "page_stride": 16 * 260}
Q8_ATTN = {**ATTN, "kv_type": B.Q8, "page_stride": 2 * 16 * 132}
READ = dict(k_pages=A, v_pages=A, n_pages=9, page_stride=2 * 16 * 132, page_size=16, n_kv_head=2, head_dim=128, kv_type=B.Q8, slots=A,
            n_tok=3, k_out=A, v_out=A, k_tok=256, v_tok=256, out_type=B.F16)
SHARED = {**ATTN, "workspace": A, "workspace_bytes": 1 << 30, "groups": A, "shared": A, "max_shared": 0, "n_group": 2}

REFUSED = {
    "qk_norm_rope": (B.QkNormRopeArgs, Q8_ROPE, [
        dict(page_stride=16 * 260 - 16), dict(page_stride=16 * 260 + 8), dict(page_stride=16 * 256), dict(kv_type=4), dict(q_type=B.Q8)]),
    "attn_paged": (B.AttnPagedArgs, Q8_ATTN, [
        dict(page_stride=2 * 16 * 132 - 16), dict(page_stride=2 * 16 * 132 + 8), dict(kv_type=4), dict(io_type=B.Q8), dict(io_type=-1),
        dict(page_size=8, page_stride=2 * 16 * 132), dict(head_dim=96), dict(k_pages=A + 8),
        dict(n_head=32768, n_kv_head=32768, n_tok=1, n_seq=1, q_tok=1 << 23, out_tok=1 << 23, page_size=65536, max_pages=1, table_stride=1,
             page_stride=1 << 40)]),
    "kv_read": (B.KvReadArgs, READ, [
        dict(head_dim=96), dict(head_dim=0), dict(n_kv_head=0), dict(n_kv_head=16385), dict(out_type=B.Q8), dict(out_type=-1),
        dict(kv_type=B.F32), dict(kv_type=4), dict(page_size=0), dict(page_size=24), dict(page_size=1 << 17), dict(n_pages=-1),
        dict(n_pages=(1 << 40) + 1), dict(page_stride=2 * 16 * 132 - 16), dict(page_stride=2 * 16 * 132 + 8),
        dict(kv_type=B.BF16, page_stride=2 * 16 * 128 - 8), dict(kv_type=B.BF16, page_stride=2 * 16 * 128 + 4), dict(k_tok=255),
        dict(v_tok=255), dict(k_tok=260), dict(v_tok=260), dict(n_tok=(1 << 30) + 1), dict(n_tok=(1 << 26) + 1), dict(k_pages=A + 8),
        dict(v_pages=A + 8), dict(slots=A + 4), dict(k_out=A + 8), dict(v_out=A + 8)]),
    "attn_shared": (B.AttnSharedArgs, SHARED, [
        dict(n_group=-1), dict(max_shared=-1), dict(groups=A + 2), dict(shared=A + 1), dict(workspace=None), dict(workspace=A + 8),
        dict(workspace_bytes=100), dict(n_group=1 << 21), dict(n_group=1 << 25), dict(head_dim=80), dict(kv_type=B.F32), dict(io_type=B.F16),
        dict(q=A + 8), dict(scale=0.0), dict(scale=INF), dict(scale=NAN), dict(max_kv=-1), dict(starts=A + 2)]),
}
NEEDED = {"qk_norm_rope": "k_pages v_pages", "attn_paged": "k_pages v_pages table", "kv_read": "k_pages v_pages slots k_out v_out",
          "attn_shared": "q out k_pages v_pages table starts kv_len groups shared workspace"}
EMPTY = {"qk_norm_rope": [dict(n_tok=0)], "attn_paged": [dict(n_tok=0)], "kv_read": [dict(n_tok=0), dict(n_tok=-1, slots=None), dict(n_pages=0)],
         "attn_shared": [dict(n_tok=0), dict(n_seq=0, groups=None)]}


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
def test_every_type_of_8_bit_calls():
    for io in (B.F32, B.F16, B.BF16):
        assert call("attn_paged", make(B.AttnPagedArgs, Q8_ATTN, io_type=io)) > 1
        assert call("kv_read", make(B.KvReadArgs, READ, out_type=io)) > 1
        assert call("qk_norm_rope", make(B.QkNormRopeArgs, Q8_ROPE, q_type=io)) > 1
        assert call("attn_shared", make(B.AttnSharedArgs, {**SHARED, **Q8_ATTN, "workspace": A, "workspace_bytes": 1 << 30}, io_type=io)) > 1
    for kv in (B.F16, B.BF16):
        assert call("kv_read", make(B.KvReadArgs, READ, kv_type=kv, page_stride=2 * 16 * 128)) > 1
    # no groups: attention without a shared prefix, for which no workspace is needed
    assert call("attn_shared", make(B.AttnSharedArgs, SHARED, n_group=0, groups=None, shared=None, workspace=None)) > 1


def test_workspace_bytes():
    def shared(**change):
        return B.lib().bonsai_p40_attn_shared_workspace_bytes(C.byref(make(B.AttnSharedArgs, {**SHARED, **change})))
    # a part is head_dim + 2 floats of each row, and there is one of the prefix and one of the own keys at least
    part = 3 * 8 * 130 * 4
    assert shared(max_kv=33, max_shared=32) == 2 * part
    n = shared(max_pages=1 << 12, table_stride=1 << 12)
    assert n > 2 * part and n % part == 0
    assert shared(head_dim=96) == 0 and shared(n_tok=0) == 0 and shared(n_group=-1) == 0
    assert shared(n_group=0, max_kv=64) == 0


def test_structs_match_the_header(tmp_path):
    """The ctypes structs have the header's sizes and offsets; attn_shared's begins with attn_paged's."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    want = {f"bonsai_p40_kv_read_args {f}": getattr(B.KvReadArgs, f).offset for f, _ in B.KvReadArgs._fields_}
    lines = [f'printf("%zu bonsai_p40_kv_read_args {f}\\n", offsetof(bonsai_p40_kv_read_args, {f}));' for f, _ in B.KvReadArgs._fields_]
    paged = {f for f, _ in B.AttnPagedArgs._fields_}
    for f, _ in B.AttnSharedArgs._fields_:
        name = "attn." + f if f in paged else f
        want[f"bonsai_p40_attn_shared_args {name}"] = getattr(B.AttnSharedArgs, f).offset
        lines.append(f'printf("%zu bonsai_p40_attn_shared_args {name}\\n", offsetof(bonsai_p40_attn_shared_args, {name}));')
    for s, cls in (("kv_read_args", B.KvReadArgs), ("attn_shared_args", B.AttnSharedArgs)):
        want[f"bonsai_p40_{s} ."] = C.sizeof(cls)
        lines.append(f'printf("%zu bonsai_p40_{s} .\\n", sizeof(bonsai_p40_{s}));')
    src, exe = tmp_path / "sizes.cpp", str(tmp_path / "sizes")
    src.write_text('#include "bonsai_p40.h"\n#include <cstdio>\nint main() {\n' + "\n".join(lines) + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(root, "include"), str(src), "-o", exe], check=True)
    got = {}
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        n, name = line.split(" ", 1)
        got[name] = int(n)
    assert got == want


def q8(n=3, kv=2, page=16, d=64):
    return B.q8_pages(n, kv, page, d, device="cpu")


def test_q8_pages():
    for n, kv, page, d in ((3, 2, 16, 64), (1, 1, 1, 64), (5, 3, 2, 128), (0, 1, 16, 64)):
        codes, scales = q8(n, kv, page, d)
        assert codes.shape == (n, kv, page, d) and scales.shape == (n, kv, page)
        assert codes.dtype is i8 and scales.dtype is torch.float32
        size = kv * page * (d + 4)
        if n > 1:
            assert codes.stride(0) == 4 * scales.stride(0) and codes.stride(0) % 16 == 0 and 0 <= codes.stride(0) - size < 16
        if n:
            assert scales.data_ptr() - codes.data_ptr() == kv * page * d


def rope(**change):
    kw = dict(q=z(5, 4, 64), k=z(5, 2, 64), v=z(5, 2, 64), q_norm=None, k_norm=None, eps=1e-6, pos=z(5, dtype=i32), inv_freq=None,
              slots=z(5, dtype=i64), k_pages=q8()[0], v_pages=q8()[0], q_out=z(5, 4, 64, dtype=f16), interleaved=False)
    return read(B.QkNormRopeArgs, B._qk_norm_rope_args(**{**kw, **change}))


def attn(**change):
    kw = dict(q=z(5, 4, 64, dtype=f16), k_pages=q8()[0], v_pages=q8()[0], table=z(2, 3, dtype=i32), starts=z(3, dtype=i32),
              kv_len=z(2, dtype=i32), out=z(5, 4, 64, dtype=f16), workspace=None, max_kv=0, scale=None)
    return read(B.AttnPagedArgs, B._attn_args(**{**kw, **change}))


def shared(**change):
    kw = dict(q=z(5, 4, 64, dtype=f16), k_pages=q8()[0], v_pages=q8()[0], table=z(2, 3, dtype=i32), starts=z(3, dtype=i32),
              kv_len=z(2, dtype=i32), groups=z(3, dtype=i32), shared=z(2, dtype=i32), out=z(5, 4, 64, dtype=f16), workspace=None, max_kv=0,
              max_shared=7, scale=None)
    return read(B.AttnSharedArgs, B._attn_shared_args(**{**kw, **change}))


def back(**change):
    kw = dict(k_pages=q8()[0], v_pages=q8()[0], slots=z(5, dtype=i64), k_out=z(5, 2, 64), v_out=z(5, 2, 64))
    return read(B.KvReadArgs, B._kv_read_args(**{**kw, **change}))


def test_wrappers_take_8_bit_pages():
    size = 2 * 16 * 68
    for a in (rope(), attn(), shared(), back(), attn(q=z(5, 4, 64), out=z(5, 4, 64))):
        assert (a.kv_type, a.n_pages, a.page_stride, a.page_size) == (B.Q8, 3, size, 16)
    assert attn(k_pages=q8(1)[0], v_pages=q8(1)[0]).page_stride == size
    assert attn(k_pages=q8(0)[0], v_pages=q8(0)[0]).n_pages == 0
    a = shared()
    assert (a.n_group, a.max_shared, a.n_seq) == (2, 7, 2)
    a = back(k_out=z(5, 3, 64)[:, :2], v_out=z(5, 2, 64))
    assert (a.n_tok, a.n_kv_head, a.head_dim, a.k_tok, a.v_tok, a.out_type) == (5, 2, 64, 192, 128, B.F32)


@pytest.mark.parametrize("pages", [
    (z(3, 2, 16, 64, dtype=i8), z(3, 2, 16, 64, dtype=i8)),                                     # no room for scales
    (q8(3, 4)[0][:, 1:3], q8(3, 4)[0][:, 1:3]),                                                 # a slice of heads: the scales are elsewhere
    (q8(3, 4)[0][:, :2], q8(3, 4)[0][:, :2]),
    (q8()[0], z(3, 2, 16, 64, dtype=f16)), (z(3, 2, 16, 64, dtype=torch.uint8),) * 2, (z(1, 2, 16, 64, dtype=i8),) * 2,
    (q8(6)[0][::2], q8(6)[0][::2])])
def test_wrappers_refuse_pages(pages):
    for f in (rope, attn, shared, back):
        with pytest.raises(ValueError):
            f(k_pages=pages[0], v_pages=pages[1])


def test_wrappers_refuse():
    for bad in (dict(groups=z(2, dtype=i32)), dict(shared=z(2)), dict(groups=z(3, dtype=i64)), dict(shared=z(3, dtype=i32)),
                dict(q=z(5, 4, 64, dtype=i8), out=z(5, 4, 64, dtype=i8)), dict(out=z(5, 4, 64))):
        with pytest.raises(ValueError):
            shared(**bad)
    for bad in (dict(slots=z(4, dtype=i64)), dict(slots=z(5, dtype=i32)), dict(k_out=z(5, 2, 32)), dict(v_out=z(4, 2, 64)),
                dict(k_out=z(5, 2, 64, dtype=f16)), dict(k_out=z(5, 2, 64, dtype=i8), v_out=z(5, 2, 64, dtype=i8)),
                dict(k_out=z(5, 64, 2).transpose(1, 2)), dict(k_out=z(5, 3, 64), v_out=z(5, 3, 64)), dict(k_out=z(5, 128))):
        with pytest.raises(ValueError):
            back(**bad)
    with pytest.raises(ValueError):                       # tensors on the device are wanted
        B.kv_read(q8()[0], q8()[0], z(5, dtype=i64), z(5, 2, 64), z(5, 2, 64))


@pytest.mark.parametrize("heads", [slice(0, 2), slice(2, 4), slice(1, 2)])
def test_wrappers_refuse_the_heads_of_one_page(heads):
    # the scales lie behind all heads' rows: where these begin does not follow from a slice of the heads
    k, v = (B.q8_pages(1, 4, 16, 64, device="cpu")[0] for _ in range(2))
    with pytest.raises(ValueError, match="8-bit pages"):
        B._pages(k[:, heads], v[:, heads], -1)
    assert B._pages(k, v, -1) == (1, 4, 16, 64, 16 * 4 * 68, B.Q8)


def test_wrappers_take_one_page_of_a_view():
    memory = torch.zeros(1, 4 * 16 * 68, dtype=i8)
    k = memory[:, :4 * 16 * 64].unflatten(1, (4, 16, 64))
    assert B._pages(k, k, -1) == (1, 4, 16, 64, 16 * 4 * 68, B.Q8)
    with pytest.raises(ValueError, match="8-bit pages"):
        B._pages(k[:, :2], k[:, :2], -1)


def test_wrappers_take_one_page_of_many():
    k, v = (B.q8_pages(5, 3, 8, 64, device="cpu")[0] for _ in range(2))
    assert B._pages(k[2:3], v[4:], -1) == (1, 3, 8, 64, 3 * 8 * 68, B.Q8)
    assert B._pages(k[:0], v[:0], -1)[0] == 0


def pages8(n, h, page=16, d=64):
    return B.q8_pages(n, h, page, d, device="cpu")[0]


@pytest.mark.parametrize("k,v", [
    (pages8(1, 2), pages8(1, 4)[:, :2]), (pages8(1, 4)[:, :2], pages8(1, 2)), (pages8(1, 2), pages8(1, 4)[:, 2:]),     # the other has its own page
    *((x, x) for x in (
        pages8(1, 4)[0, :2][None], pages8(1, 4)[0, 2:][None], pages8(3, 4)[1, :2][None], pages8(3, 2)[0][None],        # one page's stride is lost
        pages8(1, 4, 1)[0, 3:][None], torch.zeros(8, 2, 16, 64, dtype=i8)[0:1], torch.zeros(8, 2, 16, 64, dtype=i8)[7:])),   # no scales there
    (pages8(1, 2), pages8(1, 4)[0, :2][None]), (pages8(1, 2), torch.zeros(8, 2, 16, 64, dtype=i8)[0:1])])
def test_wrappers_refuse_one_page_whose_scales_are_elsewhere(k, v):
    with pytest.raises(ValueError, match="8-bit pages"):
        B._pages(k, v, -1)


def test_wrappers_take_one_page_that_is_all_there_is():
    """Its stride may be lost: memory of one page holds that page's scales."""
    for shape in ((4, 16, 64), (1, 1, 64), (3, 1, 128)):
        h, page, d = shape
        k, v = pages8(1, *shape), pages8(1, *shape)[0][None]
        want = (1, *shape, h * page * (d + 4) + -(h * page * (d + 4)) % 16, B.Q8)
        assert B._pages(k, v, -1) == B._pages(v, k, -1) == B._pages(v, v, -1) == want


def test_workspace_bytes_of_a_long_sequence_outside_the_groups():
    """The hints can say that own keys are many, though the table has room for no sequence of a prefix and so many."""
    def parts(max_kv, max_shared):
        a = make(B.AttnSharedArgs, {**SHARED, "max_pages": 1024, "table_stride": 1024, "max_kv": max_kv, "max_shared": max_shared})
        return B.lib().bonsai_p40_attn_shared_workspace_bytes(C.byref(a)) // (3 * 8 * 130 * 4)
    cap = 1024 * 16
    prefix = parts(cap, 16000) - parts(400, 16)             # (the parts of 16000 keys less those of 16, which are one)
    own = parts(16000 + 16000, 16000) - prefix - 1
    assert parts(cap, 16000) - prefix - 1 < own <= parts(16016, 16) - 1
    assert parts(1 << 40, 16000) >= parts(32000, 16000)
