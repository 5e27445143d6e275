"""Products over 16-bit weights on the GPU (grouped by expert; low-rank adapters) against plain 64-bit forms.

Tolerances, from the arithmetic alone.  A sum of n products in 32 bits is off by at most n steps of 2^-23 of the sum of the products'
magnitudes (each of its additions rounds, or truncates, by at most one such step of what has been summed).  An output rounded to
its type is off by half a step more (eps / 2 of its value).  Every element is held to that.  Over all elements the errors of the sums behave like a
random walk with a drift: at most n / 16 truncations (one for every 16 inputs that a matrix instruction takes) and sqrt(n) roundings of 2^-23 of the
result, which is what the relative 2-norm is held to, beside the outputs' half step.
"""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
pkg = load_package()
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE = {"bf16": pkg.DTYPE_BF16, "f16": pkg.DTYPE_F16, "f32": pkg.DTYPE_F32}
STEP = 2.0 ** -23
SENTINEL = -77.0


@pytest.fixture(scope="module")
def moe():
    return pkg.MoE(pkg.make_config(128, 128, 4, 1, max_tokens=4))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def hold(y, exact, slack, n, what=""):
    """y against the 64-bit result: every element within half a step of its type and `slack`, all together within the 2-norm's bound."""
    h = half_step(y.dtype)
    y = y.double()
    assert torch.isfinite(y).all(), what
    least = torch.finfo(torch.float16).smallest_normal * 2.0 ** -10 if h == 2.0 ** -11 else 0.0   # f16: the subnormals' step
    over = (y - exact).abs() - (h * (exact.abs() + slack) + slack + least)
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} elements over their bound, worst by {float(over.max()):.3e}"
    rel = float((y - exact).norm() / exact.norm().clamp_min(1e-300))
    assert rel <= h + (n / 16 + n ** 0.5) * STEP, f"{what}: rel-L2 {rel:.3e}"


class Grouped:
    """One call's inputs, laid out with strides and guards: what the call may not read is NaN, what it may not write holds a sentinel."""

    def __init__(self, sizes, K, N, dtype="bf16", out=None, layout="out_in", act="none", limit=0.0, gather=False, scatter=False, x_div=1,
                 pad=0, spare_rows=0, seed=0):
        self.sizes, self.K, self.N, self.dtype, self.out = sizes, K, N, dtype, out or dtype
        self.layout, self.act, self.limit, self.gather, self.scatter, self.x_div = layout, act, limit, gather, scatter, x_div
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt, G = DT[dtype], len(sizes)
        self.M = M = sum(sizes)
        self.rows = M + spare_rows
        NW = N * (2 if act == "swiglu" else 1)
        inner, outer = (K, NW) if layout == "out_in" else (NW, K)
        self.ld_w, self.ld_x, self.ld_y = inner + pad, K + pad, N + pad
        self.w_stride = outer * self.ld_w + 2 * pad
        w = torch.full((G * self.w_stride + 8,), float("nan"), device="cuda", dtype=dt)
        self.w = w.as_strided((G, outer, inner), (self.w_stride, self.ld_w, 1))
        for g in range(G):
            if sizes[g]:                                     # an empty group's weights stay NaN
                self.w[g] = torch.randn(outer, inner, device="cuda", generator=gen) * K ** -0.5
        self.w_all = w
        self.order = torch.cat([torch.randperm(M, device="cuda", generator=gen), torch.arange(M, self.rows, device="cuda")]).to(torch.int32)
        self.x_rows = (self.rows + x_div - 1) // x_div if gather else self.rows
        self.x_all = torch.full((self.x_rows + 1, self.ld_x), float("nan"), device="cuda", dtype=dt)
        self.x = self.x_all[:self.x_rows, :K]
        used = torch.unique(self.order[:M].long() // x_div) if gather else torch.arange(M, device="cuda")
        self.x[used] = torch.randn(len(used), K, device="cuda", generator=gen).to(dt)
        self.y_all = torch.full((self.rows + 1, self.ld_y), SENTINEL, device="cuda", dtype=DT[self.out])
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), device="cuda").to(torch.int32)

    def call(self, moe, stream=None, **kw):
        a = dict(rows=self.rows, n_groups=len(self.sizes), n_in=self.K, n_out=self.N, dtype=CODE[self.dtype], out_dtype=CODE[self.out],
                 layout=pkg.LAYOUT_OUT_IN if self.layout == "out_in" else pkg.LAYOUT_IN_OUT,
                 act=pkg.GROUPED_SWIGLU if self.act == "swiglu" else pkg.GROUPED_PLAIN, act_limit=self.limit, order=self.order.data_ptr(),
                 gather=self.gather, scatter=self.scatter, x_div=self.x_div, x_rows=self.x_rows, y_rows=self.rows, ld_x=self.ld_x,
                 ld_y=self.ld_y, ld_w=self.ld_w, w_stride=self.w_stride, stream=stream or torch.cuda.current_stream().cuda_stream)
        a.update(kw)
        moe.grouped(self.x_all.data_ptr(), self.w_all.data_ptr(), self.offsets.data_ptr(), self.y_all.data_ptr(), **a)

    def exact(self):
        """(result, bound of what 32-bit sums may be off by) in 64 bits, by sorted position"""
        y = torch.zeros(self.M, self.N, dtype=torch.float64, device="cuda")
        slack, at = torch.zeros_like(y), 0
        for g, n in enumerate(self.sizes):
            p = torch.arange(at, at + n, device="cuda")
            at += n
            if not n:
                continue
            x = self.x[self.order[p].long() // self.x_div if self.gather else p].double()
            w = self.w[g].double() if self.layout == "out_in" else self.w[g].double().T
            z, d = x @ w.T, (self.K + 1) * STEP * (x.abs() @ w.abs().T)
            if self.act == "swiglu":
                gate, up, dg, du = z[:, :self.N], z[:, self.N:], d[:, :self.N], d[:, self.N:]
                if self.limit > 0:
                    gate, up = gate.clamp(max=self.limit), up.clamp(-self.limit, self.limit)
                silu = gate * torch.sigmoid(gate)
                z = silu * up
                # |silu'| <= 1.1; the activation itself: a few roundings and an exponential, 2^-20 of its value
                d = 1.1 * dg * (up.abs() + du) + silu.abs() * du + 8 * STEP * z.abs()
            y[p], slack[p] = z, d
        return y, slack

    def check(self, what=""):
        torch.cuda.synchronize()
        exact, slack = self.exact()
        where = self.order[:self.M].long() if self.scatter else torch.arange(self.M, device="cuda")
        if self.M:
            hold(self.y_all[where, :self.N], exact, slack, self.K, what)
        rest = torch.ones(self.y_all.shape[0], dtype=torch.bool, device="cuda")
        rest[where] = False
        assert (self.y_all[rest] == SENTINEL).all(), f"{what}: rows of no group were written"
        assert (self.y_all[:, self.N:] == SENTINEL).all(), f"{what}: written past the outputs"


SIZES = {
    "one": [1], "one_of_many": [0, 0, 1, 0], "decode": [1, 0, 2, 1, 0, 0, 3, 1], "three": [3, 0, 5], "all_in_last": [0, 0, 0, 40],
    "sixteens": [16, 17, 15, 32, 33], "tiles": [128, 129, 127, 0, 1, 64, 65], "big": [300, 1, 0, 513, 255, 256, 257],
}


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("dtype, out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_grouped_against_64_bits(moe, sizes, dtype, out, act, layout):
    c = Grouped(SIZES[sizes], 264, 136, dtype, out, layout, act, 1.0 if act == "swiglu" else 0.0, pad=8, spare_rows=3)
    c.call(moe)
    c.check()


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("K, N", [(8, 8), (16, 264), (64, 128), (72, 120), (2304, 256), (5120, 8), (1032, 1400)])
@pytest.mark.parametrize("sizes", ["decode", "big"])
def test_grouped_widths(moe, K, N, sizes, layout):
    for act in ("none", "swiglu"):
        c = Grouped(SIZES[sizes], K, N, "bf16", "f32", layout, act)
        c.call(moe)
        c.check(act)


@pytest.mark.parametrize("gather, scatter", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("x_div", [1, 3, 8])
@pytest.mark.parametrize("sizes", ["decode", "three", "big"])
def test_grouped_gather_and_scatter(moe, sizes, x_div, gather, scatter):
    for layout in ("out_in", "in_out"):
        c = Grouped(SIZES[sizes], 328, 200, "bf16", "bf16", layout, "swiglu", 0.0, gather, scatter, x_div, pad=16, spare_rows=5)
        c.call(moe)
        c.check(layout)


@pytest.mark.parametrize("G, rows", [(1, 1), (1, 7), (1, 33), (1, 100), (1, 777), (1, 1300), (256, 512), (1024, 100), (1024, 3000)])
def test_grouped_many_or_one_group(moe, G, rows):
    rng = np.random.default_rng(G + rows)
    sizes = np.bincount(rng.integers(0, G, rows), minlength=G).tolist()
    c = Grouped(sizes, 520, 264, "bf16", "f32", gather=True, scatter=True, x_div=2)
    c.call(moe)
    c.check()


@pytest.mark.parametrize("rows, G, K, N", [(320, 2, 4096, 1024), (320, 2, 4096, 4096), (777, 1, 5120, 2304), (1216, 8, 4096, 4096), (3000, 16, 2304, 2048),
                                           (2400, 16, 1032, 4096), (4000, 30, 328, 4096), (6000, 8, 1032, 4096)])
def test_grouped_gathered_tiles_of_every_height(moe, rows, G, K, N):
    """Tiles of 128 to 256 rows, one item of a pair or several, parts of the reduction: rings of gathered rows of every depth."""
    rng = np.random.default_rng(rows)
    sizes = np.bincount(rng.integers(0, G, rows), minlength=G).tolist()
    for out, scatter in (("bf16", True), ("f32", False)):
        c = Grouped(sizes, K, N, "bf16", out, gather=True, scatter=scatter, x_div=4)
        c.call(moe)
        first = c.y_all.clone()
        c.check(out)
        c.call(moe)
        torch.cuda.synchronize()
        assert torch.equal(c.y_all, first)


@pytest.mark.parametrize("rows", [1, 16, 17, 200])
def test_grouped_one_group_without_offsets(moe, rows):
    c = Grouped([rows], 264, 136)
    moe.grouped(c.x_all.data_ptr(), c.w_all.data_ptr(), None, c.y_all.data_ptr(), rows, 1, 264, 136, stream=torch.cuda.current_stream().cuda_stream)
    c.check()


@pytest.mark.parametrize("H, I, tokens", [(5120, 2304, 1), (4096, 2048, 9), (6144, 2048, 70)])
def test_grouped_layer_geometries(moe, H, I, tokens):
    rng = np.random.default_rng(tokens)
    sizes = np.bincount(rng.integers(0, 16, tokens * 8), minlength=16).tolist()
    up = Grouped(sizes, H, I, act="swiglu", limit=10.0, gather=True, x_div=8)
    up.call(moe)
    up.check("gate and up")
    down = Grouped(sizes, I, H, out="f32", scatter=True)
    down.call(moe)
    down.check("down")


@pytest.mark.parametrize("sizes", ["decode", "sixteens", "big"])
def test_grouped_rows_do_not_touch_each_other(moe, sizes):
    """Infinities and NaN of a row stay in that row, those of a group's weights in that group."""
    c = Grouped(SIZES[sizes], 256, 128)
    c.call(moe)
    torch.cuda.synchronize()
    before = c.y_all.clone()
    last = c.M - 1
    c.x[0] = float("nan")
    c.x[last, 5] = float("inf")
    c.call(moe)
    torch.cuda.synchronize()
    assert torch.equal(c.y_all[1:last], before[1:last])
    assert torch.isnan(c.y_all[0, :c.N]).all() and not torch.isfinite(c.y_all[last, :c.N]).all()
    g = next(i for i, n in enumerate(c.sizes) if n)
    c.w[g] = float("nan")
    c.call(moe)
    torch.cuda.synchronize()
    assert torch.isnan(c.y_all[:c.sizes[g], :c.N]).all()
    assert torch.equal(c.y_all[max(1, c.sizes[g]):last], before[max(1, c.sizes[g]):last])


@pytest.mark.parametrize("sizes", ["decode", "big"])
def test_grouped_repeats_itself_and_runs_on_other_streams_and_in_graphs(moe, sizes):
    c = Grouped(SIZES[sizes], 1032, 264, act="swiglu", gather=True, scatter=True)
    c.call(moe)
    torch.cuda.synchronize()
    first = c.y_all.clone()
    side, other = torch.cuda.Stream(), Grouped(SIZES["tiles"], 264, 136, seed=3)
    for _ in range(3):                       # two calls of one handle in flight at once
        c.y_all.fill_(SENTINEL)
        torch.cuda.synchronize()
        c.call(moe, side.cuda_stream)
        other.call(moe)
        torch.cuda.synchronize()
        assert torch.equal(c.y_all, first)
    other.check()
    graphs = []
    for case in (c, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            case.call(moe, torch.cuda.current_stream().cuda_stream)
        case.y_all.fill_(SENTINEL)
        graphs.append(g)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(c.y_all, first)
    other.check()


def status(moe):
    return moe.stats().device_status


def test_grouped_bad_indexes_skip_their_rows_and_set_the_status(moe):
    c = Grouped(SIZES["sixteens"], 256, 128, gather=True, scatter=True)
    c.call(moe)
    torch.cuda.synchronize()
    good = c.y_all.clone()
    assert status(moe) == 0
    skipped = int(c.order[20])
    c.order[20] = 10 ** 6
    c.y_all.fill_(SENTINEL)
    c.call(moe)
    assert status(moe) == 8
    good[skipped] = SENTINEL
    assert torch.equal(c.y_all, good)
    moe.status_clear()
    for bad in ([0, 16, 33, 48, 80, 10 ** 9], [0, 16, 10, 48, 80, 113]):
        d = Grouped(SIZES["sixteens"], 256, 128)
        d.offsets.copy_(torch.tensor(bad, device="cuda", dtype=torch.int32))
        d.call(moe)
        assert status(moe) == 9
        assert (d.y_all[d.rows:] == SENTINEL).all()
        moe.status_clear()
    c = Grouped(SIZES["sixteens"], 256, 128)
    c.call(moe)
    c.check()
    assert status(moe) == 0


def test_grouped_rows_past_two_to_the_31_elements(moe):
    """Offsets that pass 32 bits: the last rows of x and y, the last groups of w."""
    K, N, G = 4096, 4096, 160                                 # w: 2.7e9 elements
    sizes = [0] * G
    sizes[0], sizes[G - 1] = 2, 3
    w = torch.zeros(G, N, K, device="cuda", dtype=torch.bfloat16)
    w[0], w[G - 1] = torch.randn(N, K, device="cuda") / 64, torch.randn(N, K, device="cuda") / 64
    x_rows = 600_000                                          # 2.5e9 elements
    x = torch.zeros(x_rows, K, device="cuda", dtype=torch.bfloat16)
    y = torch.full((x_rows, N), SENTINEL, device="cuda", dtype=torch.bfloat16)
    order = torch.tensor([x_rows - 1, 0, x_rows - 3, 5, x_rows - 2], device="cuda", dtype=torch.int32)
    x[order.long()] = torch.randn(5, K, device="cuda").to(torch.bfloat16)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), device="cuda").to(torch.int32)
    for rows in (5, 300):                                     # 300: the large calls' kernel over the same five rows
        more = torch.cat([order, torch.arange(10, 10 + rows - 5, device="cuda", dtype=torch.int32)])
        y.fill_(SENTINEL)
        moe.grouped(x.data_ptr(), w.data_ptr(), offsets.data_ptr(), y.data_ptr(), rows=rows, n_groups=G, n_in=K, n_out=N, order=more.data_ptr(),
                    gather=True, scatter=True, x_rows=x_rows, y_rows=x_rows, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        xs = x[order.long()].double()
        for p in range(5):
            m = w[0 if p < 2 else G - 1].double()
            hold(y[int(order[p])], m @ xs[p], (K + 1) * STEP * (m.abs() @ xs[p].abs()), K)
        assert (y[100] == SENTINEL).all()


# ------------------------------------------------------------------------------------------------------------
# adapters
# ------------------------------------------------------------------------------------------------------------
class Adapters:
    def __init__(self, ids, n, R, K, N, dtype="bf16", out=None, base=True, scales=True, ranks=None, pad=0, seed=0, in_place=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt, self.dtype, self.out = DT[dtype], dtype, out or dtype
        self.T, self.n, self.R, self.K, self.N, self.pad = len(ids), n, R, K, N, pad
        self.ids = torch.tensor(ids, device="cuda", dtype=torch.int32)
        nan = float("nan")
        self.x_all = torch.full((self.T + 1, K + pad), nan, device="cuda", dtype=dt)
        self.x = self.x_all[:self.T, :K]
        has = self.ids >= 0
        self.x[has] = torch.randn(int(has.sum()), K, device="cuda", generator=gen).to(dt)
        self.a_stride, self.b_stride = R * K + pad, N * R + pad
        self.a_all = torch.full((n * self.a_stride + 8,), nan, device="cuda", dtype=dt)
        self.b_all = torch.full((n * self.b_stride + 8,), nan, device="cuda", dtype=dt)
        self.a = self.a_all.as_strided((n, R, K), (self.a_stride, K, 1))
        self.b = self.b_all.as_strided((n, N, R), (self.b_stride, R, 1))
        self.rank_of = [R] * n if ranks is None else ranks
        for i in range(n):
            r = min(max(self.rank_of[i], 0), R)
            if (self.ids == i).any():
                self.a[i, :r] = torch.randn(r, K, device="cuda", generator=gen) * K ** -0.5
                self.b[i, :, :r] = torch.randn(N, r, device="cuda", generator=gen)
        self.scales = torch.rand(n, device="cuda", generator=gen) + 0.5 if scales else None
        self.ranks = None if ranks is None else torch.tensor(ranks, device="cuda", dtype=torch.int32)
        self.y_all = torch.full((self.T + 1, N + pad), SENTINEL, device="cuda", dtype=DT[self.out])
        self.base = torch.randn(self.T, N, device="cuda", generator=gen).to(DT[self.out]) if base else None
        if in_place:
            self.y_all[:self.T, :N] = self.base
        self.in_place = in_place

    def call(self, moe, stream=None):
        base, ld_base = (self.y_all, self.N + self.pad) if self.in_place else (self.base, 0)
        moe.adapters(self.x_all.data_ptr(), self.T, self.a_all.data_ptr(), self.b_all.data_ptr(), self.ids.data_ptr(), self.y_all.data_ptr(),
                     n_in=self.K, n_out=self.N, rank=self.R, n_adapters=self.n, dtype=CODE[self.dtype], out_dtype=CODE[self.out],
                     base=None if base is None else base.data_ptr(), ld_base=ld_base, scales=None if self.scales is None else self.scales.data_ptr(),
                     ranks=None if self.ranks is None else self.ranks.data_ptr(), ld_x=self.K + self.pad, ld_y=self.N + self.pad,
                     a_stride=self.a_stride, b_stride=self.b_stride, stream=stream or torch.cuda.current_stream().cuda_stream)

    def check(self, what=""):
        torch.cuda.synchronize()
        exact = self.base.double() if self.base is not None else torch.zeros(self.T, self.N, dtype=torch.float64, device="cuda")
        exact, slack = exact.clone(), torch.zeros_like(exact)
        for i in range(self.n):
            at = (self.ids == i).nonzero().squeeze(1)
            r = min(max(self.rank_of[i], 0), self.R)
            if not len(at) or not r:
                continue
            x, a, b = self.x[at].double(), self.a[i, :r].double(), self.b[i, :, :r].double()
            s = 1.0 if self.scales is None else float(self.scales[i])
            u, du = s * (x @ a.T), s * (self.K + 2) * STEP * (x.abs() @ a.abs().T)
            # the inner product as two 16-bit parts: 2^-16 of its value, and of the row's largest where f16 parts share its exponent
            du = du + 2.0 ** -16 * u.abs() + 2.0 ** -23 * u.abs().amax(1, keepdim=True)
            exact[at] += u @ b.T
            slack[at] += du @ b.abs().T + (r + 2) * STEP * (u.abs() @ b.abs().T + exact[at].abs())
        # the 2-norm: the inner product's two parts (2^-16) beside the sums
        y, h = self.y_all[:self.T, :self.N], half_step(DT[self.out])
        over = (y.double() - exact).abs() - (h * (exact.abs() + slack) + slack + 2.0 ** -24)
        assert torch.isfinite(y).all() and (over <= 0).all(), f"{what}: {int((over > 0).sum())} over, worst by {float(over.max()):.3e}"
        rel = float((y.double() - exact).norm() / exact.norm().clamp_min(1e-300))
        assert rel <= h + 2.0 ** -16 + ((self.K + self.R) / 16 + (self.K + self.R) ** 0.5) * STEP, (what, rel)
        assert (self.y_all[self.T:] == SENTINEL).all() and (self.y_all[:, self.N:] == SENTINEL).all(), what
        bare = self.ids < 0
        want = self.base[bare] if self.base is not None else torch.zeros_like(y[bare])
        assert torch.equal(y[bare], want), f"{what}: a token without an adapter is its base"


def some_ids(T, n, kind, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "runs":
        return np.sort(rng.integers(-1, n, T)).tolist()
    if kind == "none":
        return [-1] * T
    if kind == "same":
        return [n - 1] * T
    if kind == "all_different":
        return [(i * 7) % n for i in range(T)]
    return rng.integers(-1, n, T).tolist()


@pytest.mark.parametrize("T", [1, 2, 7, 16, 33, 64, 65, 200, 1000])
@pytest.mark.parametrize("kind", ["mixed", "runs", "none", "same", "all_different"])
def test_adapters_against_64_bits(moe, T, kind):
    for dtype, out, R, base in (("bf16", "bf16", 16, True), ("f16", "f16", 40, True), ("bf16", "f32", 64, False)):
        c = Adapters(some_ids(T, 70, kind), 70, R, 264, 136, dtype, out, base=base, pad=8)
        c.call(moe)
        c.check((dtype, out))


@pytest.mark.parametrize("n, T", [(511, 700), (512, 700), (3, 2048), (3, 2049), (3, 4096), (3, 4097), (511, 9000), (600, 130), (2, 65), (1, 17), (1, 64), (4, 56), (4, 55), (3, 33), (1, 431), (58, 4465), (8, 4000), (5, 300000), (600, 511), (600, 512), (600, 5000), (2047, 3000), (2048, 3000)])
@pytest.mark.parametrize("kind", ["mixed", "runs", "same"])
def test_adapters_many_tokens_and_many_adapters(moe, n, T, kind):
    """Around the sorting form's limits: 511 and 2047 adapters, segments of 2048 tokens, units of 64, 32 or 16; up to 64 tokens: 14 per adapter."""
    c = Adapters(some_ids(T, n, kind), n, 8, 40, 24, "bf16", "f32", pad=8)
    c.call(moe)
    c.check()


@pytest.mark.parametrize("R", [8, 16, 40, 64, 72, 128])
@pytest.mark.parametrize("K, N", [(8, 8), (72, 264), (1032, 1400), (2304, 512)])
@pytest.mark.parametrize("T, n", [(66, 1), (500, 7), (5000, 5)])
def test_adapters_many_tokens_each(moe, T, n, R, K, N):
    """Units of 16 tokens and more: both products on the tensor cores."""
    for dtype, out, kind in (("bf16", "bf16", "runs"), ("f16", "f32", "mixed")):
        ranks = None if dtype == "bf16" else [max(1, R - 3 * i) for i in range(n)]
        c = Adapters(some_ids(T, n, kind), n, R, K, N, dtype, out, ranks=ranks, pad=8, in_place=dtype == "f16")
        c.call(moe)
        c.check((dtype, out))


@pytest.mark.parametrize("R", [8, 16, 24, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("K, N", [(8, 8), (72, 264), (1032, 1400), (2304, 512)])
def test_adapters_widths(moe, R, K, N):
    for T in (3, 90):
        c = Adapters(some_ids(T, 5, "mixed"), 5, R, K, N, "bf16", "f32")
        c.call(moe)
        c.check(T)


@pytest.mark.parametrize("T", [1, 5, 64, 300])
def test_adapters_ranks_scales_in_place(moe, T):
    ranks = [16, 8, 0, 1, 5, 99, -3]            # over the bank's rank: the bank's; none or negative: no rows
    for dtype, out in (("bf16", "bf16"), ("f16", "f32")):
        for scales in (True, False):
            c = Adapters(some_ids(T, 7, "mixed"), 7, 16, 328, 264, dtype, out, scales=scales, ranks=ranks, in_place=True, pad=16)
            c.call(moe)
            c.check()


@pytest.mark.parametrize("H, I, T", [(5120, 2304, 1), (4096, 2048, 64), (2304, 5120, 130), (6144, 2048, 1)])
def test_adapters_layer_geometries(moe, H, I, T):
    c = Adapters(some_ids(T, 48, "mixed", 3), 48, 32, H, I, ranks=[32, 16, 8] * 16)
    c.call(moe)
    c.check()


def test_adapters_f16_products_past_its_range(moe):
    """The inner product may pass f16's largest value while the outputs do not."""
    c = Adapters([0, 1, 0], 2, 16, 256, 128, "f16", "f32", base=False)
    c.a.mul_(600.0)
    c.x.mul_(600.0)
    c.b.mul_(2.0 ** -10)
    c.call(moe)
    c.check()
    assert float((c.x[0].double() @ c.a[0].double().T).abs().max()) > 65504


@pytest.mark.parametrize("T", [9, 150])
def test_adapters_rows_do_not_touch_each_other(moe, T):
    ids = some_ids(T, 4, "mixed", 5)
    ids[0], ids[T - 1] = 1, 2
    c = Adapters(ids, 4, 24, 264, 136)
    c.call(moe)
    torch.cuda.synchronize()
    before = c.y_all.clone()
    c.x[0], c.x[T - 1, 3] = float("nan"), float("inf")
    c.call(moe)
    torch.cuda.synchronize()
    assert torch.equal(c.y_all[1:T - 1], before[1:T - 1])
    assert torch.isnan(c.y_all[0, :c.N]).all() and not torch.isfinite(c.y_all[T - 1, :c.N]).all()


def test_adapters_repeat_themselves_on_streams_and_in_graphs(moe):
    c = Adapters(some_ids(130, 9, "mixed"), 9, 32, 1032, 520, in_place=False)
    d = Adapters(some_ids(3, 9, "mixed"), 9, 16, 264, 136, seed=2)
    c.call(moe)
    torch.cuda.synchronize()
    first = c.y_all.clone()
    side = torch.cuda.Stream()
    graphs = []
    for case in (c, d):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            case.call(moe, torch.cuda.current_stream().cuda_stream)
        case.y_all.fill_(SENTINEL)
        graphs.append(g)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(c.y_all, first)
    d.check()


def test_adapters_bad_id_counts_as_none_and_sets_the_status(moe):
    ids = [0, 3, 2, 1]
    c = Adapters(ids, 3, 16, 264, 136)
    c.call(moe)
    assert status(moe) == 10
    moe.status_clear()
    c.ids[1] = -1
    c.check()


# ------------------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------------------
def test_a_layer_from_the_two_operators(moe):
    """Experts in bf16 from the library's own sort on, and a shared projection with adapters on the same tokens."""
    T, k, E, H, I = 37, 4, 12, 512, 256
    gen = torch.Generator(device="cuda").manual_seed(11)
    layer = pkg.MoE(pkg.make_config(128, 128, E, k, max_tokens=T))
    x = torch.randn(T, H, device="cuda", generator=gen).to(torch.bfloat16)
    w1 = (torch.randn(E, 2 * I, H, device="cuda", generator=gen) * H ** -0.5).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, device="cuda", generator=gen) * I ** -0.5).to(torch.bfloat16)
    ids = torch.stack([torch.randperm(E, device="cuda", generator=gen)[:k] for _ in range(T)]).to(torch.int32)
    order = torch.empty(T * k, device="cuda", dtype=torch.int32)
    offsets = torch.empty(E + 1, device="cuda", dtype=torch.int32)
    st = torch.cuda.current_stream().cuda_stream
    h = torch.empty(T * k, I, device="cuda", dtype=torch.bfloat16)
    rows = torch.empty(T * k, H, device="cuda", dtype=torch.float32)
    layer.sort_rows(ids.data_ptr(), T * k, E, order.data_ptr(), offsets.data_ptr(), st)
    layer.grouped(x.data_ptr(), w1.data_ptr(), offsets.data_ptr(), h.data_ptr(), T * k, E, H, I, act=pkg.GROUPED_SWIGLU, act_limit=2.0,
                  order=order.data_ptr(), gather=True, x_div=k, x_rows=T, stream=st)
    layer.grouped(h.data_ptr(), w2.data_ptr(), offsets.data_ptr(), rows.data_ptr(), T * k, E, I, H, out_dtype=pkg.DTYPE_F32,
                  order=order.data_ptr(), scatter=True, stream=st)
    a = (torch.randn(3, 16, H, device="cuda", generator=gen) * H ** -0.5).to(torch.bfloat16)
    b = torch.randn(3, H, 16, device="cuda", generator=gen).to(torch.bfloat16)
    ws = (torch.randn(1, H, H, device="cuda", generator=gen) * H ** -0.5).to(torch.bfloat16)
    lane = torch.tensor([0, T], device="cuda", dtype=torch.int32)
    adapter = torch.tensor(some_ids(T, 3, "mixed"), device="cuda", dtype=torch.int32)
    y = torch.empty(T, H, device="cuda", dtype=torch.float32)
    layer.grouped(x.data_ptr(), ws.data_ptr(), lane.data_ptr(), y.data_ptr(), T, 1, H, H, out_dtype=pkg.DTYPE_F32, stream=st)
    layer.adapters(x.data_ptr(), T, a.data_ptr(), b.data_ptr(), adapter.data_ptr(), y.data_ptr(), H, H, 16, 3, out_dtype=pkg.DTYPE_F32,
                   base=y.data_ptr(), stream=st)
    torch.cuda.synchronize()
    X = x.double()
    gu = torch.einsum("th,tknh->tkn", X, w1.double()[ids.long()])
    gate, up = gu[..., :I].clamp(max=2.0), gu[..., I:].clamp(-2.0, 2.0)
    hid = gate * torch.sigmoid(gate) * up
    want = torch.einsum("tki,tkhi->tkh", hid, w2.double()[ids.long()]).reshape(T * k, H)
    # h is rounded to bf16 between the products: half a step of each of its values, in the 2-norm no more than that of the result
    assert float((rows.double() - want).norm() / want.norm()) <= 2.0 ** -8
    want = X @ ws[0].double().T
    for i in range(3):
        at = (adapter == i).nonzero().squeeze(1)
        want[at] += X[at] @ a[i].double().T @ b[i].double().T
    assert float((y.double() - want).norm() / want.norm()) <= 2.0 ** -15


@pytest.mark.parametrize("T", [1, 16, 17, 64, 65, 200])
def test_shared_expert_with_adapters_in_the_layer_call(T):
    """mlxs_moe_experts_adapted with the routed rows weighted by zero: what is left is the shared expert with its adapters."""
    H, I, E, k, n, R = 512, 256, 4, 2, 5, 24
    m = pkg.MoE(pkg.make_config(H, I, E, k, bank_kind=pkg.BANK_MXFP4, act_limit=1.5, shared_expert=True, max_tokens=T))
    gen = torch.Generator(device="cuda").manual_seed(T)
    logical, _ = m.record_bytes()
    record = torch.zeros(logical, device="cuda", dtype=torch.uint8)
    record[0::7] = 127                                        # finite codes and scales of any kind
    for e in range(E):
        m.load_expert(0, e, record.data_ptr(), logical, True)
    rnd = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=gen) * std).to(torch.bfloat16)  # noqa: E731
    w1, w3, w2 = rnd(I, H, std=H ** -0.5), rnd(I, H, std=H ** -0.5), rnd(H, I, std=I ** -0.5)
    m.set_shared(0, w1.data_ptr(), w3.data_ptr(), w2.data_ptr(), True)
    ad = {"a1": rnd(n, R, H, std=H ** -0.5), "b1": rnd(n, I, R, std=0.2), "a3": rnd(n, R, H, std=H ** -0.5), "b3": rnd(n, I, R, std=0.2),
          "a2": rnd(n, R, I, std=I ** -0.5), "b2": rnd(n, H, R, std=0.2)}
    scales = torch.rand(n, device="cuda", generator=gen) + 0.5
    ranks = torch.tensor([24, 8, 16, 24, 1], device="cuda", dtype=torch.int32)
    x = rnd(T, H)
    ids = torch.zeros(T, k, device="cuda", dtype=torch.int32)
    ids[:, 1] = 1
    weights = torch.zeros(T, k, device="cuda")
    aid = torch.tensor(some_ids(T, n, "mixed", T), device="cuda", dtype=torch.int32)
    st = torch.cuda.current_stream().cuda_stream
    y, plain, none = (torch.empty(T, H, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    full = pkg.make_shared_adapters(R, n, scales=scales.data_ptr(), ranks=ranks.data_ptr(), **{c: v.data_ptr() for c, v in ad.items()})
    with pytest.raises(pkg.MlxsError) as ei:
        m.experts_adapted(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, full, aid.data_ptr(), y.data_ptr(), st)
    assert ei.value.rc == pkg.E_NOT_LOADED and "reserve_adapters" in ei.value.msg
    m.reserve_adapters()
    m.reserve_adapters()
    m.experts_adapted(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, full, aid.data_ptr(), y.data_ptr(), st)
    m.experts(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, plain.data_ptr(), st)
    m.experts_adapted(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, pkg.make_shared_adapters(R, n), aid.data_ptr(), none.data_ptr(), st)
    torch.cuda.synchronize()
    assert m.stats().device_status == 0

    # captured into a graph and replayed: the eager bits
    eager = y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.experts_adapted(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, full, aid.data_ptr(), y.data_ptr(),
                          torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        y.fill_(SENTINEL)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)

    def low_rank(v, a, b):
        out = torch.zeros(T, b.shape[1], dtype=torch.float64, device="cuda")
        for i in range(n):
            at, r = (aid == i).nonzero().squeeze(1), int(ranks[i])
            out[at] = float(scales[i]) * (v[at] @ a[i, :r].double().T @ b[i, :, :r].double().T)
        return out
    X = x.double()
    for got, on in ((y, 1.0), (plain, 0.0), (none, 0.0)):
        gate = X @ w1.double().T + on * low_rank(X, ad["a1"], ad["b1"])
        up = X @ w3.double().T + on * low_rank(X, ad["a3"], ad["b3"])
        gate, up = gate.clamp(max=1.5), up.clamp(-1.5, 1.5)
        h = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16).double()
        want = h @ w2.double().T + on * low_rank(h, ad["a2"], ad["b2"])
        # half a step of the output, and of some of h where the 32-bit sums lie next to a border (one in a hundred at most): under a whole step together
        rel = float((got.double() - want).norm() / want.norm())
        assert rel <= 2.0 ** -8 * 1.1, (T, on, rel)
    assert float((y.double() - plain.double()).norm() / plain.double().norm()) > 0.05     # the adapters do something
    bare = aid < 0
    assert float((y[bare].double() - none[bare].double()).abs().max() if bare.any() else 0.0) == 0.0


FIRST_CALLS = """
import sys, torch
from __graft_entry__ import load_package
pkg = load_package()
moe = pkg.MoE(pkg.make_config(128, 128, 4, 1, max_tokens=4))
rows, T = int(sys.argv[1]), int(sys.argv[2])
x = torch.randn(rows, 256, device="cuda").bfloat16()
w = torch.randn(2, 136, 256, device="cuda").bfloat16()
offsets = torch.tensor([0, rows // 2, rows], device="cuda", dtype=torch.int32)
y = torch.zeros(rows, 136, device="cuda", dtype=torch.bfloat16)
a, b = torch.randn(2, 64, 256, device="cuda").bfloat16(), torch.randn(2, 136, 64, device="cuda").bfloat16()
ids = (torch.arange(T, device="cuda") % 2).to(torch.int32)
z = torch.zeros(T, 136, device="cuda", dtype=torch.bfloat16)
def calls():
    s = torch.cuda.current_stream().cuda_stream
    moe.grouped(x.data_ptr(), w.data_ptr(), offsets.data_ptr(), y.data_ptr(), rows, 2, 256, 136, stream=s)
    moe.adapters(x.data_ptr(), T, a.data_ptr(), b.data_ptr(), ids.data_ptr(), z.data_ptr(), 256, 136, 64, 2, stream=s)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
assert not y.any() and not z.any()
g.replay()
torch.cuda.synchronize()
first = y.clone(), z.clone()
y.zero_(); z.zero_()
calls()
torch.cuda.synchronize()
assert torch.equal(first[0], y) and torch.equal(first[1], z) and y.any() and z.any()
assert moe.stats().device_status == 0
"""


@pytest.mark.parametrize("rows, T", [(9, 5), (200, 130), (300, 70)])
def test_a_process_whose_first_calls_are_captured(rows, T):
    """Each kernel's set-up (limits, what fits at once, tensor maps) happens inside the capture."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(rows), str(T)], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
