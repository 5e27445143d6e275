"""Two operators of the routed-MoE library as measurable cases: products grouped by expert over 16-bit weights, and the
low-rank adapters of many requests beside a shared projection.

grouped   rows sorted by group, a weight matrix per group (MoE.grouped):
            y[p] = W_g x[p]                          act "none"
            y[p] = silu(gate_g x[p]) * (up_g x[p])   act "swiglu" (gate cut from above and up from both sides at `limit` when > 0)
          for offsets[g] <= p < offsets[g + 1].  W is [groups, n_w, n_in] (layout "out_in") or [groups, n_in, n_w] ("in_out"),
          n_w = n_out, or 2 n_out with the gate's outputs first.  gather: x holds tokens and sorted position p reads row
          order[p] // top_k; scatter: position p writes row order[p] of y (order as the library's sort writes it).
adapters  y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t]; ids[t] < 0: no adapter, y[t] = base[t] (MoE.adapters).
          A is [n_adapters, rank, n_in], B [n_adapters, n_out, rank]; ranks[a] <= rank of them count.

Fields of a case are the arguments above; `rows` and `tokens` count what one call carries, `routing` says how rows spread
over the groups ("even": every group as likely, "zipf": popularity ~ rank^-1.1), `runs` how requests lie in a batch (True: each
request's tokens side by side, as in a prefill; False: interleaved, as in a decode batch), `bare` the share of tokens with no adapter.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _grouped(rows, groups, n_in, n_out, name=None, act="none", limit=0.0, dtype="bf16", out="bf16", layout="out_in", gather=False,
             scatter=False, top_k=8, routing="even"):
    c = dict(op="grouped", rows=rows, groups=groups, n_in=n_in, n_out=n_out, act=act, limit=limit, dtype=dtype, out=out, layout=layout,
             gather=gather, scatter=scatter, top_k=top_k, routing=routing)
    return c if name is None else dict(c, name=name)


def _adapters(tokens, n_adapters, rank, n_in, n_out, name=None, dtype="bf16", out="bf16", runs=False, bare=0.0, mixed=False, base=True):
    c = dict(op="adapters", tokens=tokens, n_adapters=n_adapters, rank=rank, n_in=n_in, n_out=n_out, dtype=dtype, out=out, runs=runs,
             bare=bare, mixed=mixed, base=base)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one sequence decoding: its token's eight experts, gate and up with the activation between them
        _grouped(8, 64, 5120, 2304, "experts_token", act="swiglu", limit=10.0, gather=True),
        # a full decode batch of 64 tokens over 256 experts, the down product: rows go back to assignment order in f32 for the combine
        _grouped(512, 256, 2304, 5120, "experts_batch64_down", out="f32", scatter=True),
        # a short prompt under skewed routing: a few hot experts beside experts with a row or none
        _grouped(2400, 64, 4096, 2048, "experts_chunk300_zipf", act="swiglu", gather=True, routing="zipf"),
        # prefill of 4096 tokens, gate and up
        _grouped(32768, 64, 4096, 2048, "experts_prefill4096", act="swiglu", limit=10.0, gather=True),
        # the down product of a 2048-token chunk at the widest layer
        _grouped(16384, 32, 2048, 6144, "experts_prefill2048_down", scatter=True, routing="zipf"),
        # f16 weights stored inputs first, sizes off every tile, already sorted rows
        _grouped(1003, 24, 1032, 1400, "ragged_f16_in_out", dtype="f16", out="f16", layout="in_out", routing="zipf"),
        # one group: the dense product of a shared projection over a chunk of tokens
        _grouped(777, 1, 5120, 2304, "shared_projection777", out="f32"),
        # one decoding request with an adapter: the smallest call, launches and latency
        _adapters(1, 8, 16, 5120, 2304, "adapter_token"),
        # a decode batch: 64 requests, 48 adapters of different ranks, some requests without
        _adapters(64, 48, 32, 5120, 2304, "adapters_batch64", bare=0.1, mixed=True),
        # a prefill chunk of six requests
        _adapters(8192, 6, 64, 4096, 2048, "adapters_prefill8192", runs=True, bare=0.15),
        # mixed traffic on an odd number of tokens, f16, large ranks, an f32 projection behind it
        _adapters(999, 24, 128, 2304, 5120, "adapters_mixed999_f16", dtype="f16", out="f32", mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    return rng.choice([5120, 2304, 4096, 2048, 6144, 8 * rng.randint(16, 768), 8 * rng.randint(16, 768)])


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16"])
    out = rng.choice([dtype, dtype, "f32"])
    n_in, n_out = _width(rng), _width(rng)
    if rng.random() < 0.6:
        act = rng.choice(["none", "swiglu"])
        n_w = n_out * (2 if act == "swiglu" else 1)
        # no more weights than the decode batch's bank and no more products than the largest prefill
        most_groups = min(256, 256 * 2304 * 5120 // (n_in * n_w))
        groups = _log_int(rng, 1, most_groups)
        rows = _log_int(rng, 1, min(32768, 32768 * 4096 * 4096 // (n_in * n_w)))
        return _grouped(rows, groups, n_in, n_out, act=act, limit=rng.choice([0.0, 10.0]), dtype=dtype, out=out,
                        layout=rng.choice(["out_in", "out_in", "in_out"]), gather=rng.random() < 0.5, scatter=rng.random() < 0.5,
                        top_k=rng.choice([1, 2, 8]), routing=rng.choice(["even", "zipf"]))
    return _adapters(_log_int(rng, 1, 8192), _log_int(rng, 1, 64), 8 * _log_int(rng, 1, 16), n_in, n_out, dtype=dtype, out=out,
                     runs=rng.random() < 0.5, bare=rng.choice([0.0, 0.15]), mixed=rng.random() < 0.5, base=rng.random() < 0.8)


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Rows of every group before the seed says which group gets which count: a draw that belongs to the case."""
    rng = random.Random("%(rows)d %(groups)d %(routing)s" % case)
    weights = [1.0 if case["routing"] == "even" else (1.0 + g) ** -1.1 for g in range(case["groups"])]
    sizes = [0] * case["groups"]
    for g in rng.choices(range(case["groups"]), weights, k=case["rows"]):
        sizes[g] += 1
    return sizes


def _requests(case):
    """How many tokens every adapter has (the last entry: none), again by the case alone."""
    rng = random.Random("%(tokens)d %(n_adapters)d %(bare)g" % case)
    weights = [(1.0 - case["bare"]) / case["n_adapters"]] * case["n_adapters"] + [case["bare"]]
    counts = [0] * (case["n_adapters"] + 1)
    for a in rng.choices(range(case["n_adapters"] + 1), weights, k=case["tokens"]):
        counts[a] += 1
    return counts


def _ranks(case):
    rng = random.Random("%(n_adapters)d %(rank)d" % case)
    return [rng.choice([case["rank"], max(1, case["rank"] // 2), max(1, case["rank"] // 4)]) if case["mixed"] else case["rank"]
            for _ in range(case["n_adapters"])]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen).mul_(std)

    s = {"case": case}
    if case["op"] == "grouped":
        G, K, N, M = case["groups"], case["n_in"], case["n_out"], case["rows"]
        NW = N * (2 if case["act"] == "swiglu" else 1)
        s["w"] = normal(G, NW, K, std=0.02) if case["layout"] == "out_in" else normal(G, K, NW, std=0.02)
        host = random.Random(seed)
        sizes = _sizes(case)
        host.shuffle(sizes)
        s["sizes"] = sizes
        s["offsets"] = torch.tensor([0] + sizes, device="cuda").cumsum(0).to(torch.int32)
        # a random assignment of rows to the groups, sorted as the library sorts: by group, rows of a group in their order
        group_of = torch.arange(G, device="cuda").repeat_interleave(torch.tensor(sizes, device="cuda"))
        group_of = group_of[torch.randperm(M, device="cuda", generator=gen)]
        s["order"] = torch.sort(group_of, stable=True).indices.to(torch.int32)
        s["x"] = normal((M + case["top_k"] - 1) // case["top_k"] if case["gather"] else M, K)
        s["y"] = torch.empty(M, N, device="cuda", dtype=DTYPES[case["out"]])
        return s
    T, R, K, N, n = case["tokens"], case["rank"], case["n_in"], case["n_out"], case["n_adapters"]
    s["x"] = normal(T, K)
    s["a"] = normal(n, R, K, std=K ** -0.5)
    s["b"] = normal(n, N, R, std=0.1)
    s["base"] = normal(T, N, dtype=DTYPES[case["out"]]) if case["base"] else None
    s["scales"] = torch.rand(n, device="cuda", generator=gen) + 0.5
    s["ranks"] = torch.tensor(_ranks(case), device="cuda", dtype=torch.int32)
    counts = torch.tensor(_requests(case), device="cuda")
    which = torch.cat([torch.randperm(n, device="cuda", generator=gen), torch.tensor([-1], device="cuda")])   # a seed's adapters take the counts in another order
    ids = which.repeat_interleave(counts)
    s["ids"] = (ids if case["runs"] else ids[torch.randperm(T, device="cuda", generator=gen)]).to(torch.int32)
    s["y"] = torch.empty(T, N, device="cuda", dtype=DTYPES[case["out"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from __graft_entry__ import load_package
        s["pkg"] = load_package()
        # any handle of the device serves: the operators take their own weights
        s["moe"] = s["pkg"].MoE(s["pkg"].make_config(128, 128, 256, 1, max_tokens=1))
        s["stream"] = torch.cuda.current_stream().cuda_stream
    return s


# ------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------
def _activate(gate, up, limit):
    if limit > 0:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return gate * torch.sigmoid(gate) * up


def _grouped_plain(s):
    c = s["case"]
    order = s["order"].long()
    x = s["x"].float()
    x = x[order // c["top_k"]] if c["gather"] else x
    rows, at = [], 0
    for g, n in enumerate(s["sizes"]):
        if n:
            w = s["w"][g].float()
            rows.append(x[at:at + n] @ (w.T if c["layout"] == "out_in" else w))
        at += n
    y = torch.cat(rows)
    if c["act"] == "swiglu":
        y = _activate(y[:, :c["n_out"]], y[:, c["n_out"]:], c["limit"])
    y = y.to(DTYPES[c["out"]])
    if c["scatter"]:
        return torch.empty_like(y).index_copy_(0, order, y)
    return y


def _adapters_plain(s):
    c = s["case"]
    n, R = c["n_adapters"], c["rank"]
    # all adapters' low-rank rows for every token, then the columns of its own adapter alone
    u = s["x"].float() @ s["a"].float().reshape(n * R, -1).T
    lane = torch.arange(n * R, device=u.device)
    mine = (lane // R == s["ids"].long()[:, None]) & (lane % R < s["ranks"].long()[lane // R])
    u = torch.where(mine, u * s["scales"][lane // R], 0.0)
    y = u @ s["b"].float().transpose(1, 2).reshape(n * R, -1)
    if s["base"] is not None:
        y = s["base"].float() + y
    return y.to(DTYPES[c["out"]])


def run(s):
    c = s["case"]
    if not own:
        return {"y": _grouped_plain(s) if c["op"] == "grouped" else _adapters_plain(s)}
    pkg, moe = s["pkg"], s["moe"]
    kinds = {"bf16": pkg.DTYPE_BF16, "f16": pkg.DTYPE_F16, "f32": pkg.DTYPE_F32}
    if c["op"] == "grouped":
        moe.grouped(s["x"].data_ptr(), s["w"].data_ptr(), s["offsets"].data_ptr(), s["y"].data_ptr(), rows=c["rows"], n_groups=c["groups"],
                    n_in=c["n_in"], n_out=c["n_out"], dtype=kinds[c["dtype"]], out_dtype=kinds[c["out"]],
                    layout=pkg.LAYOUT_OUT_IN if c["layout"] == "out_in" else pkg.LAYOUT_IN_OUT,
                    act=pkg.GROUPED_SWIGLU if c["act"] == "swiglu" else pkg.GROUPED_PLAIN, act_limit=c["limit"],
                    order=s["order"].data_ptr() if c["gather"] or c["scatter"] else None, gather=c["gather"], scatter=c["scatter"],
                    x_div=c["top_k"], x_rows=s["x"].shape[0], y_rows=c["rows"], stream=s["stream"])
    else:
        moe.adapters(s["x"].data_ptr(), c["tokens"], s["a"].data_ptr(), s["b"].data_ptr(), s["ids"].data_ptr(), s["y"].data_ptr(),
                     n_in=c["n_in"], n_out=c["n_out"], rank=c["rank"], n_adapters=c["n_adapters"], dtype=kinds[c["dtype"]],
                     out_dtype=kinds[c["out"]], base=s["base"].data_ptr() if c["base"] else None, scales=s["scales"].data_ptr(),
                     ranks=s["ranks"].data_ptr(), stream=s["stream"])
    return {"y": s["y"]}


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ------------------------------------------------------------------------------------------------------------
def _bytes_of(name):
    return {"bf16": 2, "f16": 2, "f32": 4}[name]


def work(case):
    wide, out = _bytes_of(case["dtype"]), _bytes_of(case["out"])
    K, N = case["n_in"], case["n_out"]
    if case["op"] == "grouped":
        M, NW = case["rows"], N * (2 if case["act"] == "swiglu" else 1)
        used = sum(1 for n in _sizes(case) if n)
        x_rows = (M + case["top_k"] - 1) // case["top_k"] if case["gather"] else M
        index = 4 * (case["groups"] + 1) + (4 * M if case["gather"] or case["scatter"] else 0)
        return {"bytes": wide * (used * NW * K + x_rows * K) + out * M * N + index, "flops": 2.0 * M * NW * K}
    T = case["tokens"]
    counts, ranks = _requests(case), sorted(_ranks(case))
    used = [n for n in counts[:-1] if n]
    # which adapters occur goes by the seed: the mean rank of the bank's adapters stands for theirs
    mean = sum(ranks) / len(ranks)
    busy = T - counts[-1]
    return {"bytes": int(wide * (len(used) * mean * (K + N) + busy * K) + out * T * N * (2 if case["base"] else 1) + 4 * T),
            "flops": 2.0 * busy * mean * (K + N)}


def exact(case, seed):
    s = _inputs(case, seed)
    K, N = case["n_in"], case["n_out"]
    if case["op"] == "grouped":
        y = torch.empty(case["rows"], N, dtype=torch.float64, device="cuda")
        ends = s["offsets"].long().tolist()
        for g in range(case["groups"]):
            at = torch.arange(ends[g], ends[g + 1], device="cuda")
            if not at.numel():
                continue
            source = torch.div(s["order"].long()[at], case["top_k"], rounding_mode="floor") if case["gather"] else at
            w = s["w"][g].double()
            z = torch.einsum("pk,nk->pn" if case["layout"] == "out_in" else "pk,kn->pn", s["x"][source].double(), w)
            if case["act"] == "swiglu":
                gate, up = z.split(N, dim=1)
                if case["limit"] > 0:
                    gate, up = torch.minimum(gate, gate.new_tensor(case["limit"])), up.clip(-case["limit"], case["limit"])
                z = gate / (1.0 + torch.exp(-gate)) * up
            y[s["order"].long()[at] if case["scatter"] else at] = z
        return {"y": y}
    y = s["base"].double() if case["base"] else torch.zeros(case["tokens"], N, dtype=torch.float64, device="cuda")
    for a in range(case["n_adapters"]):
        at = (s["ids"] == a).nonzero().squeeze(1)
        r = int(s["ranks"][a])
        u = s["x"][at].double() @ s["a"][a, :r].double().T
        y[at] += float(s["scales"][a]) * (u @ s["b"][a, :, :r].double().T)
    return {"y": y}
