"""Products over 16-bit weights on the GPU: precision of long sums and of f32 outputs, paths that the other file's sizes do not take.

Tolerances, from the arithmetic alone.
  * A matrix instruction truncates where it adds: up to four times for 16 inputs (sums of four products each), by a step of 2^-23 of what its accumulator
    holds.  With inputs of one sign an accumulator that moves on after 16 instructions holds half of its last value on average, so its value is off by
    32 steps at most; what has moved on is added with rounding, half a step for each addition, in no one direction.
  * f32 outputs of products of random signs are held to what f32 sums give: 2^-20 of the result in the 2-norm (eight steps: 16 instructions' truncations over an
    accumulator that holds half of its last value on average), or one and a half times the error of the same product in 32 bits, where that is more.
"""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from __graft_entry__ import load_package
from test_products_gpu import CODE, DT, FIRST_CALLS, SENTINEL, SIZES, STEP, Adapters, Grouped, half_step, some_ids

pytestmark = pytest.mark.gpu
pkg = load_package()


@pytest.fixture(scope="module")
def moe():
    return pkg.MoE(pkg.make_config(128, 128, 4, 1, max_tokens=4))


def stream():
    return torch.cuda.current_stream().cuda_stream


def norm_off(y, exact):
    return float((y.double() - exact).norm() / exact.norm())


def as_f32(off, off32):
    """The bound of f32 outputs: `off32` is what the same product in 32 bits is off."""
    return off <= max(2.0 ** -20, 1.5 * off32)


def one_sign_bound(terms):
    """`terms` chains of 16 instructions, or values as exact as those, added one after the other"""
    return (32 + terms ** 0.5) * STEP


def one_sign(gen, *shape, dtype):
    return (torch.rand(*shape, device="cuda", generator=gen) + 0.5).to(dtype)


def dense(moe, x, w, out, layout="out_in", act=False, gather=False):
    """x w^T (w [outputs, inputs]) by the grouped product of one group"""
    rows, K = x.shape
    N = w.shape[0] // (2 if act else 1)
    laid = w if layout == "out_in" else w.T.contiguous()
    y = torch.empty(rows, N, device="cuda", dtype=out)
    order = torch.arange(rows, device="cuda", dtype=torch.int32)
    code = {v: CODE[k] for k, v in DT.items()}
    moe.grouped(x.data_ptr(), laid.data_ptr(), None, y.data_ptr(), rows, 1, K, N, dtype=code[x.dtype], out_dtype=code[out],
                layout=pkg.LAYOUT_OUT_IN if layout == "out_in" else pkg.LAYOUT_IN_OUT, act=pkg.GROUPED_SWIGLU if act else pkg.GROUPED_PLAIN,
                order=order.data_ptr() if gather else None, gather=gather, stream=stream())
    torch.cuda.synchronize()
    return y


def activated(z):
    gate, up = z.chunk(2, dim=1)
    return gate * torch.sigmoid(gate) * up


# ------------------------------------------------------------------------------------------------------------
# up to 16 rows
# ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 16])
def test_few_rows_f32_outputs_are_as_exact_as_f32_sums(moe, rows, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    for K in (512, 2304, 6144):
        for act in (False, True):
            x = torch.randn(rows, K, device="cuda", generator=gen).to(DT[dtype])
            w = (torch.randn(512, K, device="cuda", generator=gen) * K ** -0.5).to(DT[dtype])
            z, z32 = x.double() @ w.double().T, x.float() @ w.float().T
            if act:
                z, z32 = activated(z), activated(z32)
            off, off32 = norm_off(dense(moe, x, w, torch.float32, layout, act), z), norm_off(z32, z)
            assert as_f32(off, off32), (K, act, off, off32)


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 16])
def test_few_rows_long_sums_of_one_sign(moe, rows, dtype, layout):
    """A truncated sum of one sign drifts towards zero with its length."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    for K in (6144, 65536, 262144):
        x = one_sign(gen, rows, K, dtype=DT[dtype])
        w = (one_sign(gen, 64, K, dtype=torch.float32) * (1 + torch.rand(64, 1, device="cuda", generator=gen)) / K).to(DT[dtype])
        z = x.double() @ w.double().T
        assert norm_off(dense(moe, x, w, torch.float32, layout), z) <= one_sign_bound(K / 256), K


# ------------------------------------------------------------------------------------------------------------
# tensor-core tiles
# ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [17, 64, 777])
def test_tiles_f32_outputs_are_as_exact_as_f32_sums(moe, rows, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    for K in (512, 2304, 6144):
        for act in (False, True):
            x = torch.randn(rows, K, device="cuda", generator=gen).to(DT[dtype])
            w = (torch.randn(1024, K, device="cuda", generator=gen) * K ** -0.5).to(DT[dtype])
            z, z32 = x.double() @ w.double().T, x.float() @ w.float().T
            if act:
                z, z32 = activated(z), activated(z32)
            off, off32 = norm_off(dense(moe, x, w, torch.float32, layout, act, gather=K == 2304), z), norm_off(z32, z)
            assert as_f32(off, off32), (K, act, off, off32)


@pytest.mark.parametrize("layout, act, gather", [("out_in", False, True), ("in_out", False, False), ("out_in", True, False), ("in_out", True, True)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [17, 300])
def test_tiles_long_sums_of_one_sign(moe, rows, dtype, layout, act, gather):
    """A truncated sum of one sign drifts towards zero with its length: f32 outputs, and 16-bit outputs of more inputs than one chain may take."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    N = 64
    for K, out in ((65536 + 72, "f32"), (65536 + 72, dtype), (262144, dtype)):
        x = (one_sign(gen, rows, K, dtype=torch.float32) * (1 + torch.rand(rows, 1, device="cuda", generator=gen))).to(DT[dtype])
        w = (one_sign(gen, N * (2 if act else 1), K, dtype=torch.float32) * (1 + torch.rand(N * (2 if act else 1), 1, device="cuda", generator=gen)) / K).to(DT[dtype])
        z = x.double() @ w.double().T
        z = activated(z) if act else z
        y = dense(moe, x, w, DT[out], layout, act, gather)
        # gate and up: two sums' drifts, the gate's through a slope of at most 1.1 of a value that is at least 0.73 of it
        bound = one_sign_bound(K / 1024) * (2.6 if act else 1.0)
        if out == "f32":
            assert norm_off(y, z) <= bound, (K, out)
        else:
            # an output rounds by up to half a step in no one direction: the mean of n such roundings is a drift of four of its deviations at most
            drift = float(((y.double() - z) / z).mean())
            assert abs(drift) <= bound + 4 * half_step(y.dtype) / (3 * y.numel()) ** 0.5, (K, out, drift)


# ------------------------------------------------------------------------------------------------------------
# adapters
# ------------------------------------------------------------------------------------------------------------
# tokens, adapters, rank: tiles of up to 64 tokens (16 and fewer, and more to an adapter), sorted tokens by few and by many adapters, tensor cores at ranks
# of one and two operand rows' widths, and the ranks whose rings have four slots
PATHS = [(1, 1, 16), (3, 2, 256), (40, 20, 64), (64, 48, 32), (200, 2, 8), (200, 2, 256), (700, 600, 24), (1000, 8, 40), (1000, 8, 64), (600, 8, 72), (1000, 8, 128),
         (4100, 3, 120)]


def lora(moe, x, a, b, ids, out, base=None, scales=None, ranks=None, handle_stream=None, in_place=False):
    (T, K), (n, R, _), N = x.shape, a.shape, b.shape[1]
    code = {v: CODE[k] for k, v in DT.items()}
    y = base.clone() if in_place else torch.empty(T, N, device="cuda", dtype=out)
    given = y if in_place else base
    moe.adapters(x.data_ptr(), T, a.data_ptr(), b.data_ptr(), ids.data_ptr(), y.data_ptr(), K, N, R, n, dtype=code[x.dtype], out_dtype=code[out],
                 base=None if given is None else given.data_ptr(), scales=None if scales is None else scales.data_ptr(),
                 ranks=None if ranks is None else ranks.data_ptr(), stream=handle_stream or stream())
    torch.cuda.synchronize()
    return y


def lora_plain(x, a, b, ids, base, scales, wide):
    y = torch.zeros(x.shape[0], b.shape[1], device="cuda", dtype=wide) if base is None else base.to(wide)
    y = y.clone()
    for i in range(a.shape[0]):
        at = (ids == i).nonzero().squeeze(1)
        if len(at):
            s = 1.0 if scales is None else scales[i].to(wide)
            y[at] += (x[at].to(wide) @ a[i].to(wide).T * s) @ b[i].to(wide).T
    return y


def adapters_off(moe, T, n, R, K, N, dtype, based, seed=0):
    """(the call's error, that of the same products in 32 bits)"""
    gen = torch.Generator(device="cuda").manual_seed(seed + T)
    x = torch.randn(T, K, device="cuda", generator=gen).to(DT[dtype])
    a = (torch.randn(n, R, K, device="cuda", generator=gen) * K ** -0.5).to(DT[dtype])
    b = (torch.randn(n, N, R, device="cuda", generator=gen) * 0.1).to(DT[dtype])
    ids = torch.randint(0, n, (T,), device="cuda", generator=gen).to(torch.int32)
    scales = torch.rand(n, device="cuda", generator=gen) + 0.5
    base = torch.randn(T, N, device="cuda", generator=gen) if based else None
    y = lora(moe, x, a, b, ids, torch.float32, base, scales, in_place=based)
    exact = lora_plain(x, a, b, ids, base, scales, torch.float64)
    return norm_off(y, exact), norm_off(lora_plain(x, a, b, ids, base, scales, torch.float32), exact)


@pytest.mark.parametrize("based", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R", PATHS)
def test_adapters_f32_outputs_are_as_exact_as_f32_sums(moe, T, n, R, dtype, based):
    """Few inputs: what is kept of the inner product decides."""
    off, off32 = adapters_off(moe, T, n, R, 264, 136, dtype, based)
    assert as_f32(off, off32), (off, off32)


SUMS = [(1, 1, 16, 5120, 2304), (16, 1, 16, 6144, 512), (40, 2, 64, 5120, 520), (64, 1, 32, 6144, 520), (300, 2, 256, 6144, 520), (4000, 8, 16, 5120, 2304), (3000, 600, 24, 4096, 520)]
SUMS_TENSOR = [(1000, 8, 64, 5120, 2304), (1000, 8, 72, 6144, 264), (4100, 3, 120, 1024, 520), (1000, 8, 128, 5120, 520), (8192, 6, 64, 5120, 520), (4100, 300, 40, 2304, 264)]


def check_sums(moe, T, n, R, K, N, dtype, based):
    off, off32 = adapters_off(moe, T, n, R, K, N, dtype, based)
    assert as_f32(off, off32), (off, off32)


def check_one_sign(moe, T, n, R, K, dtype):
    """Inner products of one sign drift together, and the outputs with them; 2^-20 beside it for the outer product."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    x, a = one_sign(gen, T, K, dtype=DT[dtype]), (one_sign(gen, n, R, K, dtype=torch.float32) / K).to(DT[dtype])
    b = torch.randn(n, 136, R, device="cuda", generator=gen).to(DT[dtype])
    ids = torch.randint(0, n, (T,), device="cuda", generator=gen).to(torch.int32)
    off = norm_off(lora(moe, x, a, b, ids, torch.float32), lora_plain(x, a, b, ids, None, None, torch.float64))
    assert off <= one_sign_bound(K / 256) + 2.0 ** -20, off


@pytest.mark.parametrize("based", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R, K, N", SUMS)
def test_adapters_inner_sums(moe, T, n, R, K, N, dtype, based):
    check_sums(moe, T, n, R, K, N, dtype, based)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R, K", [(1, 1, 16, 262144), (40, 1, 64, 262144), (300, 2, 200, 65536 + 8), (1000, 2, 16, 262144), (3000, 600, 8, 16384)])
def test_adapters_long_inner_sums_of_one_sign(moe, T, n, R, K, dtype):
    check_one_sign(moe, T, n, R, K, dtype)


@pytest.mark.parametrize("based", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R, K, N", SUMS_TENSOR)
def test_adapters_inner_sums_on_the_tensor_cores(moe, T, n, R, K, N, dtype, based):
    check_sums(moe, T, n, R, K, N, dtype, based)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R, K", [(1000, 2, 64, 262144), (4100, 2, 64, 65536 + 8), (4100, 300, 40, 16384), (2048, 16, 128, 24576)])
def test_adapters_long_inner_sums_of_one_sign_on_the_tensor_cores(moe, T, n, R, K, dtype):
    check_one_sign(moe, T, n, R, K, dtype)


@pytest.mark.parametrize("dtype, out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("T, n, R", [(3, 2, 16), (50, 2, 32), (200, 2, 24), (1000, 8, 64)])
def test_adapters_infinite_scale(moe, T, n, R, dtype, out):
    """An infinite scale makes infinities of an adapter of rank one, of the product's sign, and stays in its tokens."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 128, device="cuda", generator=gen).to(DT[dtype])
    a, b = torch.randn(n, R, 128, device="cuda", generator=gen).to(DT[dtype]), torch.randn(n, 72, R, device="cuda", generator=gen).to(DT[dtype])
    b[b == 0] = 1
    ids = (torch.arange(T, device="cuda") % n).to(torch.int32)
    scales, ranks = torch.ones(n, device="cuda"), torch.ones(n, device="cuda", dtype=torch.int32)
    finite = lora(moe, x, a, b, ids, DT[out], scales=scales, ranks=ranks)
    assert torch.isfinite(finite).all()
    scales[1] = float("inf")
    y = lora(moe, x, a, b, ids, DT[out], scales=scales, ranks=ranks)
    mine = ids == 1
    u = (x[mine].double() @ a[1, 0].double())[:, None] * b[1, :, 0].double()
    assert (u != 0).all() and torch.equal(y[mine].double(), u.sign() * float("inf"))
    assert torch.equal(y[~mine], finite[~mine])


# ------------------------------------------------------------------------------------------------------------
# several host threads
# ------------------------------------------------------------------------------------------------------------
def in_threads(works):
    """Each of `works` in a thread of its own, all at once; what they raised."""
    raised, ready = [], threading.Barrier(len(works))

    def run(work):
        try:
            torch.cuda.set_device(0)
            ready.wait()
            work()
        except Exception as e:                           # noqa: BLE001
            raised.append(e)
    threads = [threading.Thread(target=run, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return raised


@pytest.mark.parametrize("shapes", [((200, 2, 256), (200, 2, 8)), ((4000, 2, 64), (4000, 2, 128)), ((40, 2, 256), (40, 2, 16))])
def test_adapters_of_two_handles_on_two_threads(shapes):
    """The same kernel with another amount of shared memory from each thread."""
    def calls(T, n, R):
        m = pkg.MoE(pkg.make_config(128, 128, 4, 1, max_tokens=4))
        gen = torch.Generator(device="cuda").manual_seed(R)
        x = torch.randn(T, 64, device="cuda", generator=gen).to(torch.bfloat16)
        a, b = torch.randn(n, R, 64, device="cuda", generator=gen).to(torch.bfloat16), torch.randn(n, 64, R, device="cuda", generator=gen).to(torch.bfloat16)
        ids = (torch.arange(T, device="cuda") % n).to(torch.int32)
        want = lora(m, x, a, b, ids, torch.bfloat16)
        y = torch.empty_like(want)
        st = torch.cuda.Stream()
        torch.cuda.synchronize()

        def work():
            for i in range(20000):
                m.adapters(x.data_ptr(), T, a.data_ptr(), b.data_ptr(), ids.data_ptr(), y.data_ptr(), 64, 64, R, n, stream=st.cuda_stream)
                if i % 500 == 499:
                    st.synchronize()
            assert torch.equal(y, want)
        return work
    assert in_threads([calls(*s) for s in shapes]) == []


@pytest.mark.parametrize("T", [1, 20, 300])
@pytest.mark.parametrize("bank", ["BANK_EXL3_K3_MUL1", "BANK_MXFP4"])
def test_layers_of_two_handles_on_two_threads(bank, T):
    """Handles of two geometries: the streaming kernels, the front, the router's logits and the dispatch take other amounts of shared memory."""
    def calls(H, I, E):
        m = pkg.MoE(pkg.make_config(H, I, E, 2, bank_kind=getattr(pkg, bank), max_tokens=T))
        gen = torch.Generator(device="cuda").manual_seed(H)
        logical, _ = m.record_bytes()
        record = torch.zeros(logical, device="cuda", dtype=torch.uint8)
        record[1::7] = 60
        for e in range(E):
            m.load_expert(0, e, record.data_ptr(), logical, True)
        w = torch.randn(E, H, device="cuda", generator=gen).to(torch.bfloat16)
        m.set_router_weight(0, w.data_ptr(), True)
        x = torch.randn(T, H, device="cuda", generator=gen).to(torch.bfloat16)
        y = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        m.forward_x(0, x.data_ptr(), T, y.data_ptr(), st.cuda_stream)
        torch.cuda.synchronize()
        want = y.clone()

        def work():
            for i in range(30000 if T == 1 else 5000):
                m.forward_x(0, x.data_ptr(), T, y.data_ptr(), st.cuda_stream)
                if i % 100 == 99:
                    st.synchronize()
            assert torch.equal(y.view(torch.int16), want.view(torch.int16)) and m.stats().device_status == 0
        return work
    assert in_threads([calls(512, 256, 8), calls(5120, 512, 64)]) == []


# ------------------------------------------------------------------------------------------------------------
# waits that run out
# ------------------------------------------------------------------------------------------------------------
@pytest.fixture
def waiting():
    """A handle of the test's own, whose waits are short while a ring stage is left out of every producer's."""
    m = pkg.MoE(pkg.make_config(128, 128, 4, 1, max_tokens=4))
    yield m
    m.debug_wait(0, 0)
    m.close()


def runs_out(m, call, y, stage, writes_nothing=True):
    """`call` writes y: it returns, reports, stores nothing that waited, and the call after it is right."""
    y.fill_(SENTINEL)
    call()
    torch.cuda.synchronize()
    good = y.clone()
    assert m.stats().device_status == 0 and not (good == SENTINEL).any()
    y.fill_(SENTINEL)
    m.debug_wait(poll_limit=300, withhold_stage=stage)
    call()
    torch.cuda.synchronize()
    m.debug_wait(0, 0)
    assert m.stats().device_status in (2, 3)
    left = y == SENTINEL
    assert left.all() if writes_nothing else torch.equal(y[~left], good[~left]) and left.any()
    m.status_clear()
    assert m.stats().device_status == 0
    call()
    torch.cuda.synchronize()
    assert m.stats().device_status == 0 and torch.equal(y, good)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("rows, K, N, stage", [(64, 5120, 2304, 1), (64, 5120, 2304, 5), (300, 5120, 2304, 2), (3000, 1024, 1024, 1)])
def test_tiles_whose_wait_runs_out(waiting, rows, K, N, stage, out, gather):
    """Parts of the reduction over a cluster (64 and 300 rows), and pairs that walk the tiles."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, K, device="cuda", generator=gen).to(torch.bfloat16)
    w = (torch.randn(N, K, device="cuda", generator=gen) * K ** -0.5).to(torch.bfloat16)
    y = torch.empty(rows, N, device="cuda", dtype=DT[out])
    order = torch.arange(rows, device="cuda", dtype=torch.int32)
    runs_out(waiting, lambda: waiting.grouped(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), rows, 1, K, N, out_dtype=CODE[out],
                                              order=order.data_ptr(), gather=gather, stream=stream()), y, stage)


@pytest.mark.parametrize("T, n, R, stage", [(1000, 8, 64, 1), (1000, 8, 128, 7), (200, 1, 128, 1), (3000, 2, 64, 35)])
@pytest.mark.parametrize("dtype, out", [("bf16", "f32"), ("f16", "f16")])
def test_adapters_whose_wait_runs_out(waiting, T, n, R, stage, dtype, out):
    """Stages of the inner product, and of the outer one (the last case: 46 units, clusters of two, 32 stages and then eight)."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 4096, device="cuda", generator=gen).to(DT[dtype])
    a = (torch.randn(n, R, 4096, device="cuda", generator=gen) / 64).to(DT[dtype])
    b = torch.randn(n, 2048, R, device="cuda", generator=gen).to(DT[dtype])
    ids = (torch.arange(T, device="cuda") % n).to(torch.int32)
    y = torch.empty(T, 2048, device="cuda", dtype=DT[out])
    runs_out(waiting, lambda: waiting.adapters(x.data_ptr(), T, a.data_ptr(), b.data_ptr(), ids.data_ptr(), y.data_ptr(), 4096, 2048, R, n,
                                               dtype=CODE[dtype], out_dtype=CODE[out], stream=stream()), y, stage, writes_nothing=stage < 35)


def test_a_failed_run_is_not_hidden_by_what_a_call_answers_as_documented(waiting):
    """The status word is sticky: an adapter id that counts as none before, or after, a wait that ran out; a slot id taken for another."""
    x, w = torch.randn(64, 1024, device="cuda").to(torch.bfloat16), torch.randn(512, 1024, device="cuda").to(torch.bfloat16)
    a, b = torch.randn(1, 8, 1024, device="cuda").to(torch.bfloat16), torch.randn(1, 512, 8, device="cuda").to(torch.bfloat16)
    y = torch.zeros(64, 512, device="cuda", dtype=torch.bfloat16)
    ids = torch.ones(64, device="cuda", dtype=torch.int32)
    slots = torch.tensor([0, 99, 1], device="cuda", dtype=torch.int32)
    order, offsets = torch.zeros(3, device="cuda", dtype=torch.int32), torch.zeros(5, device="cuda", dtype=torch.int32)

    def bad_id():
        waiting.adapters(x.data_ptr(), 64, a.data_ptr(), b.data_ptr(), ids.data_ptr(), y.data_ptr(), 1024, 512, 8, 1, stream=stream())

    def bad_slot():
        waiting.sort_rows(slots.data_ptr(), 3, 4, order.data_ptr(), offsets.data_ptr(), stream())

    def lost_wait():
        waiting.debug_wait(poll_limit=300, withhold_stage=1)
        waiting.grouped(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), 64, 1, 1024, 512, stream=stream())
        waiting.debug_wait(0, 0)

    def status_after(*calls):
        waiting.status_clear()
        for c in calls:
            c()
        torch.cuda.synchronize()
        return waiting.stats().device_status
    assert status_after(bad_id) == 10 and status_after(bad_slot) == 1 and status_after(lost_wait) in (2, 3)
    assert status_after(bad_id, lost_wait) in (2, 3) and status_after(lost_wait, bad_id) in (2, 3)
    assert status_after(bad_slot, lost_wait) in (2, 3) and status_after(lost_wait, bad_slot) in (2, 3)
    assert status_after(bad_id, bad_slot) == 1 and status_after(bad_slot, bad_id) == 1
    waiting.status_clear()


# ------------------------------------------------------------------------------------------------------------
# kernels that the other file's sizes and types do not take
# ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("sizes", ["one", "decode", "all_in_last", "sixteens", "big"])
def test_grouped_f16_with_f32_outputs(moe, sizes, act, layout):
    c = Grouped(SIZES[sizes], 264, 136, "f16", "f32", layout, act, 1.0 if act == "swiglu" else 0.0, gather=sizes == "decode", scatter=True, x_div=2, pad=8, spare_rows=3)
    c.call(moe)
    c.check()


@pytest.mark.parametrize("dtype, out", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("sizes", ["sixteens", "big"])
def test_grouped_of_more_inputs_than_a_chain(moe, sizes, dtype, out):
    """Odd lengths of the last chain and stage, with running sums for 16-bit outputs (f16)."""
    for K, layout, act in ((8200, "out_in", "none"), (8648, "in_out", "swiglu"), (9216, "out_in", "swiglu")):
        c = Grouped(SIZES[sizes], K, 72, dtype, out, layout, act, gather=K == 8648, scatter=True, pad=8, spare_rows=2)
        c.call(moe)
        first = c.y_all.clone()
        c.check(K)
        c.call(moe)
        torch.cuda.synchronize()
        assert torch.equal(c.y_all, first)


@pytest.mark.parametrize("R", [40, 64, 72, 120, 128])
@pytest.mark.parametrize("K, N", [(8, 8), (72, 264), (1032, 1400), (2304, 512)])
@pytest.mark.parametrize("T, n", [(500, 7), (5000, 5)])
def test_adapters_on_the_tensor_cores_of_the_layer_calls_types(moe, T, n, R, K, N):
    for dtype, out, in_place in (("bf16", "f32", True), ("f16", "f16", False)):
        ranks = [max(1, R - 3 * i) for i in range(n)] if in_place else None
        c = Adapters(some_ids(T, n, "mixed" if in_place else "runs"), n, R, K, N, dtype, out, ranks=ranks, pad=8, in_place=in_place)
        c.call(moe)
        first = c.y_all.clone()
        c.check((dtype, out))
        if not in_place:
            c.call(moe)
            torch.cuda.synchronize()
            assert torch.equal(c.y_all, first)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R, K", [(5, 2, 16, 20008), (50, 1, 64, 33000), (300, 2, 256, 20480), (700, 600, 24, 16392), (1000, 8, 64, 24584)])
def test_adapters_of_long_inputs_with_16_bit_outputs(moe, T, n, R, K, dtype):
    c = Adapters(some_ids(T, n, "mixed"), n, R, K, 72, dtype, pad=8)
    c.call(moe)
    c.check()


def test_adapters_of_two_ranks_in_one_graph(moe):
    """One kernel with two amounts of shared memory, captured side by side and replayed; eager calls of other ranks in between."""
    calls = [Adapters(some_ids(T, n, "mixed", T), n, R, 520, 264, "bf16", out, ranks=[R, 1, R - 4], seed=R)
             for T, n, R, out in ((1000, 3, 64, "f32"), (1000, 3, 128, "f32"), (40, 3, 256, "bf16"), (40, 3, 8, "bf16"), (500, 3, 16, "bf16"), (500, 3, 256, "bf16"))]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in calls:
            c.call(moe, stream())
    for c in calls:
        c.y_all.fill_(SENTINEL)
    for _ in range(2):
        g.replay()
        Adapters(some_ids(300, 3, "mixed"), 3, 72, 520, 264, "bf16", "f32").call(moe)
        torch.cuda.synchronize()
        for c in calls:
            c.check()


@pytest.mark.parametrize("rows, T", [(400, 400), (1000, 900)])
def test_a_process_whose_first_calls_of_the_tensor_core_kernels_are_captured(rows, T):
    """400 tokens of two adapters, rank 64: the adapters' tensor map and its query of the clusters that fit happen inside the capture."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(rows), str(T)], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("T, R", [(400, 64), (900, 128), (300, 200)])
def test_shared_expert_with_adapters_of_many_tokens(T, R):
    """The layer call where its adapters take the tensor cores (bf16 inputs, f32 rows in place): what the routed rows, weighted by zero, leave."""
    H, I, E, k, n = 512, 384, 4, 2, 3
    m = pkg.MoE(pkg.make_config(H, I, E, k, bank_kind=pkg.BANK_MXFP4, act_limit=1.5, shared_expert=True, max_tokens=T))
    gen = torch.Generator(device="cuda").manual_seed(T)
    logical, _ = m.record_bytes()
    record = torch.zeros(logical, device="cuda", dtype=torch.uint8)
    for e in range(E):
        m.load_expert(0, e, record.data_ptr(), logical, True)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(torch.bfloat16)
    w1, w3, w2 = rnd(I, H, std=H ** -0.5), rnd(I, H, std=H ** -0.5), rnd(H, I, std=I ** -0.5)
    m.set_shared(0, w1.data_ptr(), w3.data_ptr(), w2.data_ptr(), True)
    m.reserve_adapters()
    ad = {"a1": rnd(n, R, H, std=H ** -0.5), "b1": rnd(n, I, R, std=0.1), "a3": rnd(n, R, H, std=H ** -0.5), "b3": rnd(n, I, R, std=0.1),
          "a2": rnd(n, R, I, std=I ** -0.5), "b2": rnd(n, H, R, std=0.1)}
    x, y = rnd(T, H), torch.empty(T, H, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(T, k, device="cuda", dtype=torch.int32)
    ids[:, 1] = 1
    weights, aid = torch.zeros(T, k, device="cuda"), torch.tensor(some_ids(T, n, "mixed", T), device="cuda", dtype=torch.int32)
    full = pkg.make_shared_adapters(R, n, **{c: v.data_ptr() for c, v in ad.items()})
    m.experts_adapted(0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, full, aid.data_ptr(), y.data_ptr(), stream())
    torch.cuda.synchronize()
    assert m.stats().device_status == 0

    def linear(v, w, a, b):
        return lora_plain(v, a, b, aid, v @ w.double().T, None, torch.float64)
    gate, up = linear(x.double(), w1, ad["a1"], ad["b1"]).clamp(max=1.5), linear(x.double(), w3, ad["a3"], ad["b3"]).clamp(-1.5, 1.5)
    h = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16).double()
    # half a step of the output, and of those values of h whose f32 sums lie next to a rounding border (one in a hundred at most)
    assert norm_off(y, linear(h, w2, ad["a2"], ad["b2"])) <= 2.0 ** -8 * 1.1
    m.close()


# ------------------------------------------------------------------------------------------------------------
# the largest calls, and calls behind copies
# ------------------------------------------------------------------------------------------------------------
def test_grouped_most_rows_and_groups(moe):
    """2^22 sorted positions of 1024 groups, gathered and scattered."""
    gen = torch.Generator().manual_seed(1)
    cuts = torch.sort(torch.randint(0, 2 ** 22 + 1, (1023,), generator=gen)).values.tolist()
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [2 ** 22])]
    c = Grouped(sizes, 16, 8, "bf16", "f32", gather=True, scatter=True, x_div=8)
    c.call(moe)
    c.check()
    assert moe.stats().device_status == 0


@pytest.mark.parametrize("n", [3, 511, 2047, 5000])
def test_adapters_most_tokens(moe, n):
    T = 2 ** 22
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(T, 8, device="cuda", generator=gen).to(torch.bfloat16)
    a, b = torch.randn(n, 8, 8, device="cuda", generator=gen).to(torch.bfloat16), torch.randn(n, 8, 8, device="cuda", generator=gen).to(torch.bfloat16)
    ids = torch.randint(-1, n, (T,), device="cuda", generator=gen).to(torch.int32)
    y = lora(moe, x, a, b, ids, torch.float32)
    at = torch.randint(0, T, (20000,), device="cuda", generator=gen)
    at[:3] = torch.tensor([0, T - 1, T - 2], device="cuda")
    i = ids[at].long().clamp(min=0)
    u = torch.einsum("tk,trk->tr", x[at].double(), a[i].double())
    want = torch.einsum("tr,tor->to", u, b[i].double()) * (ids[at] >= 0)[:, None]
    assert norm_off(y[at], want) <= 2.0 ** -20 and (y[ids < 0] == 0).all()
    assert moe.stats().device_status == 0


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("K, N", [(262144, 8), (8, 262144)])
def test_grouped_longest_and_widest(moe, K, N, layout, rows):
    for act in ("none", "swiglu"):
        c = Grouped([rows], K, N, "bf16", "f32", layout, act)
        c.call(moe)
        c.check(act)


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("K, N", [(262144, 8), (8, 262144)])
def test_adapters_longest_and_widest(moe, K, N, T):
    for R in (16, 64, 256):
        c = Adapters([0] * T, 1, R, K, N, "bf16", "f32")
        c.call(moe)
        c.check(R)


def test_products_behind_copies_in_a_graph(moe):
    """A call's launch begins under the one before it; behind a copy or a memset of a graph it waits as any other."""
    g40, g9 = Grouped([20, 0, 20], 264, 136, gather=True), Grouped([4, 5], 264, 136)
    ad = Adapters(some_ids(500, 3, "mixed"), 3, 64, 264, 136, "bf16", "f32", in_place=True)
    few = Adapters(some_ids(9, 3, "mixed"), 3, 16, 264, 136)
    calls = (g40, g9, ad, few)
    sources = [c.x_all.clone() for c in calls]
    base = ad.y_all.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c, s in zip(calls, sources):
            c.x_all.copy_(s)
            if c is ad:
                c.y_all.copy_(base)
            c.call(moe, stream())
    for k in range(3):
        for c, s in zip(calls, sources):
            s.mul_(-1.0)                                 # the rows of this replay
            c.x_all.zero_()
            if c is not ad:
                c.y_all.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        for c in calls:
            c.check(k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T, n, R", [(700, 600, 256), (3000, 2047, 136), (200, 3, 136), (64, 2, 248), (9, 2, 136)])
def test_adapters_of_ranks_above_128_with_f32_outputs(moe, T, n, R, dtype):
    """The most shared memory (three parts, tables of many adapters), the first rank whose outer products are rounded, ranks of their own."""
    c = Adapters(some_ids(T, n, "mixed"), n, R, 328, 136, dtype, "f32", ranks=[R - 8 * (i % 9) for i in range(n)], pad=8)
    c.call(moe)
    c.check()
    off, off32 = adapters_off(moe, T, min(n, 20), R, 1032, 136, dtype, False)
    assert as_f32(off, off32), (off, off32)
