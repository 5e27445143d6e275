"""The products over 16-bit weights without a GPU: every refusal is decided before a device is touched."""
import ctypes as C

import pytest

from __graft_entry__ import load_package

pkg = load_package()
P = 1 << 20      # an aligned address that no refused call reads


def grouped(handle=None, x=P, w=P, offsets=P, order=P, y=P, **kw):
    f = dict(struct_size=C.sizeof(pkg.GroupedDesc), dtype=0, out_dtype=0, layout=0, act=0, act_limit=0.0, n_groups=4, n_in=256, n_out=128,
             rows=16, row_flags=0, x_div=1, x_rows=16, y_rows=16, ld_x=0, ld_y=0, ld_w=0, w_stride=0)
    f.update(kw)
    return pkg.lib().mlxs_moe_grouped(handle, C.byref(pkg.GroupedDesc(**f)), x, w, offsets, order, y, None)


def adapters(handle=None, x=P, a=P, b=P, ids=P, scales=None, ranks=None, base=P, y=P, **kw):
    f = dict(struct_size=C.sizeof(pkg.AdaptersDesc), dtype=0, out_dtype=0, n_in=256, n_out=128, rank=16, n_adapters=3, tokens=5, ld_x=0,
             ld_base=0, ld_y=0, a_stride=0, b_stride=0)
    f.update(kw)
    return pkg.lib().mlxs_moe_adapters(handle, C.byref(pkg.AdaptersDesc(**f)), x, a, b, ids, scales, ranks, base, y, None)


def test_descriptors_match_the_header_layout():
    assert C.sizeof(pkg.GroupedDesc) == 14 * 4 + 4 * 8
    assert C.sizeof(pkg.AdaptersDesc) == 8 * 4 + 5 * 8


@pytest.mark.parametrize("kw, rc, word", [
    (dict(struct_size=8), pkg.E_CONFIG, "struct_size"), (dict(dtype=2), pkg.E_CONFIG, "dtype"), (dict(out_dtype=1), pkg.E_CONFIG, "out_dtype"),
    (dict(layout=2), pkg.E_CONFIG, "layout"), (dict(act=2), pkg.E_CONFIG, "act"), (dict(act=1, act_limit=-1.0), pkg.E_CONFIG, "act_limit"),
    (dict(act=1, act_limit=float("nan")), pkg.E_CONFIG, "act_limit"), (dict(act=1, act_limit=float("inf")), pkg.E_CONFIG, "act_limit"),
    (dict(act_limit=1.0), pkg.E_CONFIG, "act_limit"), (dict(n_groups=0), pkg.E_CONFIG, "n_groups"), (dict(n_groups=1025), pkg.E_CONFIG, "n_groups"),
    (dict(n_in=0), pkg.E_CONFIG, "n_in"), (dict(n_in=100), pkg.E_CONFIG, "n_in"), (dict(n_out=12), pkg.E_CONFIG, "n_out"),
    (dict(n_out=1 << 20), pkg.E_CONFIG, "n_out"), (dict(rows=(1 << 22) + 1, x_rows=1 << 22, y_rows=1 << 22), pkg.E_TOO_MANY_TOKENS, "rows"),
    (dict(row_flags=4), pkg.E_CONFIG, "row_flags"), (dict(x_rows=15), pkg.E_ARG, "x_rows"), (dict(y_rows=15), pkg.E_ARG, "y_rows"),
    (dict(row_flags=1, x_div=0), pkg.E_ARG, "x_div"), (dict(row_flags=1, x_rows=0), pkg.E_ARG, "x_rows"),
    (dict(row_flags=2, y_rows=0), pkg.E_ARG, "y_rows"), (dict(ld_x=248), pkg.E_ARG, "ld_x"), (dict(ld_x=260), pkg.E_ARG, "ld_x"),
    (dict(ld_y=120), pkg.E_ARG, "ld_y"), (dict(ld_w=128), pkg.E_ARG, "ld_w"), (dict(layout=1, ld_w=120), pkg.E_ARG, "ld_w"),
    (dict(w_stride=256 * 127), pkg.E_ARG, "w_stride"), (dict(w_stride=1 << 40), pkg.E_ARG, "w_stride"), (dict(x=None), pkg.E_ARG, "x_dev"),
    (dict(w=P + 8), pkg.E_ARG, "w_dev"), (dict(y=P + 2), pkg.E_ARG, "y_dev"), (dict(x=P + 8), pkg.E_ARG, "x_dev"),
    (dict(offsets=P + 2), pkg.E_ARG, "offsets_dev"), (dict(offsets=None), pkg.E_ARG, "offsets_dev"),
    (dict(offsets=None, n_groups=1), pkg.E_ARG, "null handle"),
    (dict(row_flags=1, order=None), pkg.E_ARG, "order_dev"), (dict(row_flags=2, order=P + 1), pkg.E_ARG, "order_dev"),
    (dict(), pkg.E_ARG, "null handle"), (dict(rows=0), pkg.E_ARG, "null handle"),
])
def test_grouped_refuses_by_name(kw, rc, word):
    assert grouped(**kw) == rc, pkg.last_error()
    assert pkg.last_error().startswith("grouped: ") and word in pkg.last_error()


@pytest.mark.parametrize("kw, rc, word", [
    (dict(struct_size=8), pkg.E_CONFIG, "struct_size"), (dict(dtype=2, out_dtype=2), pkg.E_CONFIG, "dtype"), (dict(out_dtype=1), pkg.E_CONFIG, "out_dtype"),
    (dict(n_in=4), pkg.E_CONFIG, "n_in"), (dict(n_out=0), pkg.E_CONFIG, "n_out"), (dict(rank=0), pkg.E_CONFIG, "rank"),
    (dict(rank=12), pkg.E_CONFIG, "rank"), (dict(rank=264), pkg.E_CONFIG, "rank"), (dict(n_adapters=0), pkg.E_CONFIG, "n_adapters"),
    (dict(tokens=(1 << 22) + 1), pkg.E_TOO_MANY_TOKENS, "tokens"), (dict(ld_x=128), pkg.E_ARG, "ld_x"), (dict(ld_base=132), pkg.E_ARG, "ld_base"),
    (dict(ld_y=64), pkg.E_ARG, "ld_y"), (dict(a_stride=256 * 8), pkg.E_ARG, "a_stride"), (dict(b_stride=4), pkg.E_ARG, "b_stride"),
    (dict(x=None), pkg.E_ARG, "x_dev"), (dict(a=P + 4), pkg.E_ARG, "a_dev"), (dict(b=P + 4), pkg.E_ARG, "b_dev"), (dict(ids=P + 1), pkg.E_ARG, "ids_dev"),
    (dict(y=None), pkg.E_ARG, "y_dev"), (dict(base=P + 8), pkg.E_ARG, "base_dev"), (dict(scales=P + 1), pkg.E_ARG, "scales_dev"),
    (dict(ranks=P + 2), pkg.E_ARG, "ranks_dev"), (dict(ld_base=136), pkg.E_ARG, "in place"), (dict(), pkg.E_ARG, "null handle"),
    (dict(tokens=0), pkg.E_ARG, "null handle"),
])
def test_adapters_refuse_by_name(kw, rc, word):
    assert adapters(**kw) == rc, pkg.last_error()
    assert pkg.last_error().startswith("adapters: ") and word in pkg.last_error()


@pytest.mark.parametrize("kw, rc, word", [
    (dict(struct_size=8), pkg.E_CONFIG, "struct_size"), (dict(rank=4), pkg.E_CONFIG, "rank"), (dict(rank=512), pkg.E_CONFIG, "rank"),
    (dict(n_adapters=0), pkg.E_CONFIG, "n_adapters"), (dict(a1=None), pkg.E_ARG, "a1_dev"), (dict(b3=None), pkg.E_ARG, "a3_dev"),
    (dict(a2=P + 8), pkg.E_ARG, "a2_dev"), (dict(scales=P + 2), pkg.E_ARG, "scales_dev"), (dict(ranks=P + 1), pkg.E_ARG, "ranks_dev"),
    (dict(ids=None), pkg.E_ARG, "adapter_ids_dev"), (dict(), pkg.E_ARG, "null handle"),
])
def test_experts_adapted_refuses_by_name(kw, rc, word):
    f = dict(struct_size=C.sizeof(pkg.SharedAdapters), rank=16, n_adapters=2, a1=P, b1=P, a3=P, b3=P, a2=P, b2=P, scales=P, ranks=P)
    ids = kw.pop("ids", P)
    f.update(kw)
    assert pkg.lib().mlxs_moe_experts_adapted(None, 0, P, P, P, 3, C.byref(pkg.SharedAdapters(**f)), ids, P, None) == rc, pkg.last_error()
    assert pkg.last_error().startswith("experts_adapted: ") and word in pkg.last_error()


def test_null_descriptors_are_refused():
    assert C.sizeof(pkg.SharedAdapters) == 16 + 8 * 8
    assert pkg.lib().mlxs_moe_experts_adapted(None, 0, P, P, P, 3, None, P, P, None) == pkg.E_ARG
    assert pkg.lib().mlxs_moe_reserve_adapters(None) == pkg.E_ARG
    L = pkg.lib()
    assert L.mlxs_moe_grouped(None, None, P, P, P, P, P, None) == pkg.E_ARG
    assert L.mlxs_moe_adapters(None, None, P, P, P, P, None, None, P, P, None) == pkg.E_ARG
