"""The token mixers' kernels are of the hot path, whose scratch, spills and budgets
test_kernel_resources.py looks at."""
from test_kernel_resources import kr, pytestmark, rows  # noqa: F401


def test_the_mixers_are_on_the_hot_path(rows):  # noqa: F811
    families = {f: [r for r in rows if kr.family(r) == f]
                for f in ("qk_norm_rope_kernel", "attn_kernel", "attn_join_kernel", "gdn_step_kernel", "gdn_prep_kernel",
                          "gdn_scan_kernel")}
    for f, built in families.items():
        assert built and all(kr.is_hot_path(r) for r in built), f
        assert not any(r["scratch"] or r["vgpr_spill"] or r["sgpr_spill"] for r in built), f


def test_attention_keeps_its_waves(rows):  # noqa: F811
    # heads of 64 and 128 share a CU's registers between two workgroups of 4 waves (rows; 128 with three terms of
    # fp32 queries: one), heads of 256 have one wave a SIMD
    for r in rows:
        if kr.family(r) != "attn_kernel":
            continue
        d, terms, keys = r["name"].split("<")[1].split(">")[0].split(", ")[1:4]
        if keys == "false" and d in ("64", "128") and (d, terms) != ("128", "3"):
            assert r["vgpr"] + r["agpr"] <= 256, r["name"]
