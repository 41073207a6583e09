"""The measured cases of the row operators: group norm with an activation, rows kept in 8 bits, and the 8-bit product that reads them.

``own = False``: the operators from elementary torch operations; ``own = True``: the framework's entry points (``ogl_amd.ops``).  Both take what
``prepare`` gives and return the same outputs.  ``exact`` states each operator in 64 bits.
"""
import math

import torch

own = False

F32, BF16, F16 = "float32", "bfloat16", "float16"
VERTICES, FEATURES, HIDDEN = 232965, 602, 600        # the Reddit-shaped stream of the benchmark
BLOCK = 62500                                        # input rows of one of its 512-seed blocks

QMAX = {"int8": 127.0, "e4m3": 448.0}
AMAX_FLOOR = 2.0 ** -80


# ------------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # hidden rows of one 32-seed step (32 x 26 destinations, 32 wide): what latency decides
        dict(name="norm_rows_small", op="norm", train=True, b=832, l=1, c=32, g=4, dtype=F32, act="silu"),
        # the input rows of one 512-seed block, 600 wide, forward and backward of a train step
        dict(name="norm_rows_block", op="norm", train=True, b=BLOCK, l=1, c=HIDDEN, g=30, dtype=F32, act="gelu"),
        # serving on maps of positions (channels last): 8 of 64 x 64, 32 groups of 10 channels
        dict(name="norm_map_serve", op="norm", train=False, b=8, l=4096, c=320, g=32, dtype=BF16, act="silu"),
        # training on long ones: 4 of 128 x 128
        dict(name="norm_map_train", op="norm", train=True, b=4, l=16384, c=512, g=32, dtype=BF16, act="silu"),
        # one snapshot's few new vertices into a small table, and the table read back
        dict(name="rows_append", op="rows", fmt="int8", n=64, m=57, width=FEATURES, group=0, dtype=F32, slots="ids"),
        # one decoding step of 32 sequences: a token of 8 heads of 128 each, written where a page table says
        dict(name="rows_token", op="rows", fmt="e4m3", n=512, m=32, width=1024, group=128, dtype=F16, slots="ids"),
        # the whole vertex table as it is loaded, then gathered by a block's ids
        dict(name="rows_table", op="rows", fmt="int8", n=VERTICES, m=VERTICES, width=FEATURES, group=0, dtype=F32, slots="start"),
        # a long prompt's heads into a cache whose slots come in any order, some of them twice
        dict(name="rows_heads", op="rows", fmt="e4m3", n=131072, m=131072, width=1024, group=128, dtype=BF16, slots="ids"),
        # the projection of one vertex that has just arrived
        dict(name="linear_vertex", op="linear", m=1, k=FEATURES, n=HIDDEN, dtype=F32, relu=True, rows=0),
        # a decoding step of 16 sequences through a wide layer: the weight's bytes decide
        dict(name="linear_tokens", op="linear", m=16, k=4096, n=12288, dtype=BF16, relu=False, rows=0),
        # fc_pool over one block's rows, gathered from the vertex table
        dict(name="linear_block", op="linear", m=BLOCK, k=FEATURES, n=HIDDEN, dtype=F32, relu=True, rows=VERTICES),
        # a prompt through a wide layer: the matrix units decide
        dict(name="linear_prompt", op="linear", m=8192, k=4096, n=8192, dtype=BF16, relu=False, rows=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rows", "linear"])
    if op == "norm":
        g = rng.choice([1, 2, 3, 4, 7, 8, 16, 30, 32])
        c = g * max(8, _log(rng, 8, 640) // g)
        l = 1 if rng.random() < 0.5 else _log(rng, 2, 16384)
        b = min(_log(rng, 1, 62500), max(1, 32_000_000 // (l * c)))
        return dict(op="norm", train=rng.random() < 0.6, b=b, l=l, c=c, g=g, dtype=rng.choice([F32, BF16, F16]), act=rng.choice(["silu", "gelu", "none"]))
    if op == "rows":
        width = _log(rng, 9, 4096)
        n = min(_log(rng, 16, 232965), 130_000_000 // width)
        m = max(1, int(n * rng.uniform(0.1, 1.0)))
        return dict(op="rows", fmt=rng.choice(["int8", "e4m3"]), n=n, m=m, width=width, group=rng.choice([0, 16, 64, 96, 128]),
                    dtype=rng.choice([F32, BF16, F16]), slots=rng.choice(["start", "ids"]))
    m, k, n = _log(rng, 1, 62500), _log(rng, 17, 4096), _log(rng, 3, 8192)
    m = max(1, min(m, 250_000_000_000 // (2 * k * n), 60_000_000 // n))
    return dict(op="linear", m=m, k=k, n=n, dtype=rng.choice([F32, BF16, F16]), relu=rng.random() < 0.5, rows=rng.choice([0, _log(rng, 16, 100_000)]))


def work(case):
    size = 4 if case["dtype"] == F32 else 2
    if case["op"] == "norm":
        x = case["b"] * case["l"] * case["c"]
        return dict(bytes=x * size * (5 if case["train"] else 2) + 4 * case["c"] * (4 if case["train"] else 2), flops=x * (40 if case["train"] else 12))
    if case["op"] == "rows":
        n, m, w = case["n"], case["m"], case["width"]
        g = 1 if case["group"] == 0 else -(-w // case["group"])
        return dict(bytes=m * (w * (size + 1) + 4 * g) + n * (w * (size + 1) + 4 * g) + 8 * n + (8 * m if case["slots"] == "ids" else 0), flops=4 * (m + n) * w)
    m, k, n = case["m"], case["k"], case["n"]
    return dict(bytes=m * k + n * k + 4 * m + 8 * n + m * n * size + (8 * m if case["rows"] else 0), flops=2 * m * n * k)


# ------------------------------------------------------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(n, width, gen):
    """int8 rows as the framework keeps them: whole rows of 64 bytes, zeros behind the last column."""
    codes = torch.zeros((n, -(-width // 64) * 64), dtype=torch.int8, device="cuda")
    codes[:, :width] = torch.randn((n, width), generator=gen, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)
    return codes


def prepare(case, seed):
    gen = _gen(seed)
    dtype = getattr(torch, case["dtype"])
    s = dict(case=case)
    if case["op"] == "norm":
        shape = (case["b"], case["c"]) if case["l"] == 1 else (case["b"], case["l"], case["c"])
        s["x"] = torch.randn(shape, generator=gen, device="cuda").mul_(1.5).add_(0.3).to(dtype)
        s["weight"] = torch.rand(case["c"], generator=gen, device="cuda") + 0.5
        s["bias"] = torch.randn(case["c"], generator=gen, device="cuda") * 0.2
        if case["train"]:
            s["dy"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
        return s
    if case["op"] == "rows":
        n, m, w = case["n"], case["m"], case["width"]
        group = case["group"] or w
        # rows of different sizes, as activations and features have them
        s["x"] = (torch.randn((m, w), generator=gen, device="cuda") * torch.exp(torch.randn((m, 1), generator=gen, device="cuda"))).to(dtype)
        s["group"] = group
        s["codes"] = torch.zeros((n, -(-w // 64) * 64), dtype=torch.int8, device="cuda")
        s["scales"] = torch.rand((n, -(-w // group)), generator=gen, device="cuda") * 0.01
        s["codes"][:, :w] = torch.randint(-100, 101, (n, w), generator=gen, device="cuda", dtype=torch.int8)
        if case["fmt"] == "e4m3":
            s["codes"] = s["codes"].float().to(torch.float8_e4m3fn)
        s["slots"], s["start"] = None, 0
        if case["slots"] == "ids":
            slots = torch.randperm(n, generator=gen, device="cuda")[:m]
            again = torch.rand(m, generator=gen, device="cuda")
            slots = torch.where(again < 0.03, slots[torch.randint(0, m, (m,), generator=gen, device="cuda")], slots)      # some slots twice
            s["slots"] = torch.where(again > 0.99, torch.full_like(slots, -1), slots).contiguous()                      # some rows are padding
        s["rows"] = torch.randperm(n, generator=gen, device="cuda")
        if own:
            from ogl_amd import ops
            s["cache"] = ops.QuantRows(s["codes"], s["scales"], w, group)
        return s
    m, k, n = case["m"], case["k"], case["n"]
    have = case["rows"] or m
    s["x"], s["w"] = _codes(have, k, gen), _codes(n, k, gen)
    s["sx"] = (torch.rand((have, 1), generator=gen, device="cuda") + 0.5) * 0.02
    s["sw"] = (torch.rand((n, 1), generator=gen, device="cuda") + 0.5) * 0.002
    s["bias"] = torch.randn(n, generator=gen, device="cuda")
    s["rows"] = torch.randint(0, have, (m,), generator=gen, device="cuda") if case["rows"] else None
    if own:
        from ogl_amd import ops
        s["qx"], s["qw"] = ops.QuantRows(s["x"], s["sx"], k), ops.QuantRows(s["w"], s["sw"], k)
    return s


# ------------------------------------------------------------------------------------------------------------- the plain forms
def _act(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * 0.7071067811865476))
    return torch.relu(z) if act == "relu" else z


def _act_slope(z, act):
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    return (z > 0).float() if act == "relu" else torch.ones_like(z)


def _norm_plain(s):
    case = s["case"]
    b, l, c, g = case["b"], case["l"], case["c"], case["g"]
    with torch.no_grad():
        x = s["x"].float().reshape(b, l, g, c // g)
        mean = x.mean((1, 3), keepdim=True)
        h = x - mean
        rstd = 1 / torch.sqrt((h * h).mean((1, 3), keepdim=True) + 1e-5)
        h = h * rstd
        w = s["weight"].reshape(1, 1, g, c // g)
        z = h * w + s["bias"].reshape(1, 1, g, c // g)
        y = _act(z, case["act"]).reshape(s["x"].shape).to(s["x"].dtype)
        if not case["train"]:
            return y
        dz = s["dy"].float().reshape(b, l, g, c // g) * _act_slope(z, case["act"])
        dzh = dz * h
        dw, db = dzh.sum((0, 1)).reshape(c), dz.sum((0, 1)).reshape(c)
        dh = dz * w
        dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - h * (dzh * w).mean((1, 3), keepdim=True))
        return [y, dx.reshape(s["x"].shape).to(s["x"].dtype), dw, db]


def _scales_of(x, fmt, group):
    """x [m, width] in 64 bits -> (x and its scales by group, both with the ragged last group filled up): a scale is the float32 nearest amax / Q."""
    m, w = x.shape
    groups = -(-w // group)
    x = torch.nn.functional.pad(x, (0, groups * group - w)).reshape(m, groups, group)
    amax = x.abs().amax(2).clamp(min=AMAX_FLOOR)
    scale = (amax / QMAX[fmt]).float()
    return x, torch.where(torch.isfinite(amax), scale, torch.full_like(scale, math.nan))


def _round_e4m3(t):
    """To the nearest e4m3 value, ties to even, in 64 bits: 3 bits behind the leading one, none below 2^-9."""
    exponent = torch.frexp(t)[1] - 1
    step = torch.ldexp(torch.ones_like(t), exponent.clamp(min=-6) - 3)
    return torch.round(t / step) * step


def _rows_plain(s):
    case = s["case"]
    n, m, w, group = case["n"], case["m"], case["width"], s["group"]
    x, scale = _scales_of(s["x"].double(), case["fmt"], group)
    t = x / scale.double().unsqueeze(2)                         # in 64 bits: values next to a border
    t = torch.round(t) if case["fmt"] == "int8" else _round_e4m3(t)
    t = torch.where(torch.isfinite(t), t, torch.zeros_like(t))
    codes = t.reshape(m, -1)[:, :w].float().to(s["codes"].dtype)
    if s["slots"] is None:
        s["codes"][s["start"]:s["start"] + m, :w] = codes
        s["scales"][s["start"]:s["start"] + m] = scale
    else:
        at = torch.arange(m, device="cuda")
        slot = torch.where((s["slots"] >= 0) & (s["slots"] < n), s["slots"], torch.full_like(s["slots"], n))
        last = torch.full((n + 1,), -1, device="cuda", dtype=torch.int64).scatter_reduce_(0, slot, at, "amax")[:n]       # of a slot's rows the last
        hit = last >= 0
        hit1, last = hit.unsqueeze(1), last.clamp(min=0)
        s["codes"][:, :w] = torch.where(hit1, codes.float()[last], s["codes"][:, :w].float()).to(s["codes"].dtype)
        s["scales"].copy_(torch.where(hit1, scale[last], s["scales"]))
    rows = s["rows"]
    values = s["codes"].float()[rows][:, :w] * torch.repeat_interleave(s["scales"][rows], group, dim=1)[:, :w]
    return values.to(s["x"].dtype)


def _linear_plain(s):
    case = s["case"]
    x, sx = s["x"], s["sx"]
    if s["rows"] is not None:
        x, sx = x[s["rows"]], sx[s["rows"]]
    y = (x.float() @ s["w"].float().t()) * (sx * s["sw"].t()) + s["bias"]
    return (torch.relu(y) if case["relu"] else y).to(getattr(torch, case["dtype"]))


# ---------------------------------------------------------------------------------------------------------- the framework's own
def _own(s):
    from ogl_amd import ops
    case = s["case"]
    if case["op"] == "norm":
        if not case["train"]:
            with torch.no_grad():
                return ops.group_norm(s["x"], case["g"], s["weight"], s["bias"], activation=None if case["act"] == "none" else case["act"])
        y = ops.group_norm(s["x"], case["g"], s["weight"], s["bias"], activation=None if case["act"] == "none" else case["act"])
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])]
    if case["op"] == "rows":
        ops.quant_rows_write(s["cache"], s["x"], slots=s["slots"], start=s["start"])
        return ops.quant_rows_read(s["cache"], s["rows"], dtype=s["x"].dtype)
    return ops.linear_int8(s["qx"], s["qw"], s["bias"], relu=case["relu"], x_rows=s["rows"], dtype=getattr(torch, case["dtype"]))


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm_plain, "rows": _rows_plain, "linear": _linear_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _nearest(t, grid):
    """The value of the sorted `grid` nearest to each of t >= 0, of two at the same distance the one at the even place."""
    hi = torch.searchsorted(grid, t).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - t, t - grid[lo]
    take = torch.where(up == down, hi % 2 == 0, up < down)
    return torch.where(take, grid[hi], grid[lo])


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] == "norm":
        b, c, g = case["b"], case["c"], case["g"]
        leaves = [s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias")]
        with torch.set_grad_enabled(case["train"]):
            x = leaves[0].reshape(b, -1, g, c // g).transpose(1, 2).reshape(b, g, -1)
            var, mean = torch.var_mean(x, dim=2, correction=0, keepdim=True)
            h = ((x - mean) * torch.rsqrt(var + 1e-5)).reshape(b, g, -1, c // g).transpose(1, 2).reshape(b, -1, c)
            z = h * leaves[1] + leaves[2]
            y = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "none": lambda v: v}[case["act"]](z)
            y = y.reshape(s["x"].shape)
            if not case["train"]:
                return y
            return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double())]
    if case["op"] == "rows":
        n, m, w, group, fmt = case["n"], case["m"], case["width"], s["group"], case["fmt"]
        grid = torch.arange(128, device="cuda", dtype=torch.float64)
        if fmt == "e4m3":
            grid = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        old = s["codes"].double()[:, :w]
        out = torch.empty((n, w), dtype=torch.float64, device="cuda")
        # later rows of a slot replace earlier ones: the rows sorted by (slot, place), the last of each slot
        at = torch.arange(m, device="cuda")
        slot = s["slots"] if s["slots"] is not None else at + s["start"]
        order = torch.argsort(slot, stable=True)
        sorted_slot = slot[order]
        ends = torch.ones(m, dtype=torch.bool, device="cuda")
        ends[:-1] = sorted_slot[:-1] != sorted_slot[1:]
        rows, to = order[ends & (sorted_slot >= 0)], sorted_slot[ends & (sorted_slot >= 0)]
        for lo in range(0, w, group):
            hi = min(w, lo + group)
            out[:, lo:hi] = old[:, lo:hi] * s["scales"][:, lo // group].double().unsqueeze(1)
            x = s["x"][rows, lo:hi].double()
            scale = (x.abs().amax(1, keepdim=True).clamp(min=AMAX_FLOOR) / QMAX[fmt]).float().double()
            out[to, lo:hi] = torch.sign(x) * _nearest(x.abs() / scale, grid) * scale
        return out[s["rows"]]
    x, sx = s["x"], s["sx"].double()
    if s["rows"] is not None:
        x, sx = x[s["rows"]], sx[s["rows"]]
    y = torch.mm(x[:, :case["k"]].double(), s["w"][:, :case["k"]].double().t())
    y = y * sx * s["sw"].double().reshape(1, -1) + s["bias"].double()
    return y.clamp(min=0) if case["relu"] else y
