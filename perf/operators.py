"""Timing cases of the operators over a model's columns: the normalisation of columns, the routing of columns to experts,
the distillation loss against a sparse teacher and the product of an 8-bit dense matrix with a sparse one.

A dense matrix of the library is column-major: an n x m matrix is a torch tensor of shape (m, n) here, one row of the
tensor per column. A sparse matrix is CSC (ir, jc, values). run() computes a case either with elementary torch
operations (own = False) or with the library's entry points (own = True), on the same state.

norm          h = x + r, y = w * h / sqrt(mean(h^2) + eps), and y in e4m3 with one scale per group of rows
norm_grad     the gradients of y (and of h) with respect to x and w
route         the topk experts of every column as a CSC matrix of weights, and how often each was taken
route_grad    the gradient of the weights with respect to the scores
distill       tau^2 * KL(softmax(teacher / tau) || softmax(z / tau)) per column and its gradient with respect to z
distill_grad  that gradient from a kept log-sum
q8            A * S with A in e4m3 and scales
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
KINDS = {"softmax": 0, "sigmoid": 1}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-5


def listed():
    return [
        # one new token of a served model: residual added, the normalised column in 8 bits for the products that follow
        {"name": "norm_token", "op": "norm", "n": 4096, "m": 1, "type": "bf16", "res": True, "y": False, "group": 128},
        # a prompt of 16384 tokens, served: residual, 8 bits with a scale per 128 rows
        {"name": "norm_prompt", "op": "norm", "n": 8192, "m": 16384, "type": "bf16", "res": True, "y": False, "group": 128},
        # a factor model's columns of an odd height in single precision, with both outputs
        {"name": "norm_odd", "op": "norm", "n": 1001, "m": 7777, "type": "f32", "res": False, "y": True, "group": 0},
        # the backward pass of a training step, with the gradient that arrives over the residual
        {"name": "norm_train", "op": "norm_grad", "n": 4096, "m": 16384, "type": "bf16", "res": True},
        # a handful of new tokens over 256 experts in 8 groups, sigmoid scores with a balancing bias
        {"name": "route_tokens", "op": "route", "e": 256, "m": 8, "type": "f32", "kind": "sigmoid", "bias": True, "groups": 8,
         "topgroups": 4, "k": 8, "renorm": True},
        # the same over a long prompt
        {"name": "route_prompt", "op": "route", "e": 256, "m": 65536, "type": "bf16", "kind": "sigmoid", "bias": True, "groups": 8,
         "topgroups": 4, "k": 8, "renorm": True},
        # a training step's forward pass over an odd number of experts: plain softmax weights, no groups
        {"name": "route_train", "op": "route", "e": 60, "m": 32768, "type": "f32", "kind": "softmax", "bias": False, "groups": 1,
         "topgroups": 1, "k": 4, "renorm": False},
        # its backward pass over 128 experts
        {"name": "route_back", "op": "route_grad", "e": 128, "m": 32768, "type": "bf16", "kind": "softmax", "bias": False, "groups": 1,
         "topgroups": 1, "k": 6, "renorm": False},
        # a few columns over an odd vocabulary in single precision: one column has to use the whole card
        {"name": "distill_few", "op": "distill", "v": 100003, "m": 5, "type": "f32", "k": 20, "tau": 2.0, "ragged": True},
        # a training batch of 4096 tokens: loss and gradient in one call
        {"name": "distill_batch", "op": "distill", "v": 131072, "m": 4096, "type": "bf16", "k": 64, "tau": 1.0, "ragged": False},
        # the backward pass alone, from the kept log-sums, teachers of different lengths and empty columns
        {"name": "distill_back", "op": "distill_grad", "v": 50001, "m": 2048, "type": "f16", "k": 100, "tau": 1.5, "ragged": True},
        # embedding bags over a table of 200000 columns in 8 bits, column lengths from a power law
        {"name": "q8_bags", "op": "q8", "n": 1024, "rows": 200000, "cols": 50000, "mean": 40, "law": "pareto", "group": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "route", "route_grad", "distill", "distill_grad", "q8"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("norm", "norm_grad"):
        n = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        m = _log(rng, 1, max(2, min(65536, (1 << 26) // n)))
        case = {"op": op, "n": n, "m": m, "type": kind, "res": rng.random() < 0.7}
        if op == "norm":
            case["y"] = rng.random() < 0.5
            case["group"] = rng.choice([0, 32, 64, 128]) if rng.random() < 0.7 or not case["y"] else -1
        return case
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 4, 8])
        e = groups * max(4, _log(rng, 8, 512) // groups)
        topgroups = rng.randint(1, groups)
        k = rng.randint(1, min(16, topgroups * (e // groups)))
        m = _log(rng, 1, min(65536, (1 << 24) // e))
        return {"op": op, "e": e, "m": m, "type": kind, "kind": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5,
                "groups": groups, "topgroups": topgroups, "k": k, "renorm": rng.random() < 0.5}
    if op in ("distill", "distill_grad"):
        v = _log(rng, 1000, 262144)
        m = _log(rng, 1, max(2, min(16384, (1 << 28) // v)))
        return {"op": op, "v": v, "m": m, "type": kind, "k": _log(rng, 2, 256), "tau": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "ragged": rng.random() < 0.7}
    n = _log(rng, 16, 2048)
    if rng.random() < 0.7:
        n = max(16, n // 16 * 16)
    mean = _log(rng, 2, 64)
    cols = _log(rng, 8, max(16, min(100000, (1 << 30) // (n * mean))))
    return {"op": "q8", "n": n, "rows": _log(rng, 1000, 200000), "cols": cols, "mean": mean, "law": rng.choice(["pareto", "even"]),
            "group": rng.choice([0, 32, 64, 128])}


# ---------------------------------------------------------------- inputs

def _ngroups(n, group):
    return 1 if group == 0 else -(-n // group)


def _csc(lengths):
    jc = torch.zeros(lengths.numel() + 1, dtype=torch.int32, device="cuda")
    jc[1:] = torch.cumsum(lengths, 0)
    ic = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), lengths)
    return jc, ic


def _distinct_rows(g, lengths, jc, ic, rows):
    """Different rows within every column: an arithmetic sequence from a random start, with a random step that is odd and
    small enough not to come round."""
    longest = max(1, int(lengths.max()))
    start = torch.randint(0, rows, (lengths.numel(),), generator=g, device="cuda")
    step = torch.randint(1, max(2, rows // longest), (lengths.numel(),), generator=g, device="cuda")
    at = torch.arange(ic.numel(), device="cuda") - jc[:-1].long()[ic]
    return ((start[ic] + at * step[ic]) % rows).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    op = case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op in ("norm", "norm_grad"):
        n, m, t = case["n"], case["m"], DTYPES[case["type"]]
        s["w"] = 1 + 0.1 * normal(n)
        if op == "norm":
            s["X"] = (2 * normal(m, n)).to(t)
            s["R"] = normal(m, n).to(t) if case["res"] else None
            s["H"] = torch.empty(m, n, dtype=t, device="cuda") if case["res"] else None
            s["Y"] = torch.empty(m, n, dtype=t, device="cuda") if case["y"] else None
            s["Q"] = s["scales"] = None
            if case["group"] >= 0:
                s["Q"] = torch.empty(m, n, dtype=torch.float8_e4m3fn, device="cuda")
                s["scales"] = torch.empty(m, _ngroups(n, case["group"]), device="cuda")
        else:
            s["H"] = (2 * normal(m, n)).to(t)
            s["dY"] = normal(m, n).to(t)
            s["dH"] = normal(m, n).to(t) if case["res"] else None
            s["dX"] = torch.empty(m, n, dtype=t, device="cuda")
            s["dw"] = torch.empty(n, device="cuda")
    elif op in ("route", "route_grad"):
        e, m, k, t = case["e"], case["m"], case["k"], DTYPES[case["type"]]
        Z = 1.5 * normal(m, e)
        if m > 4:
            Z[-(m // 16 + 1):] = -math.inf                 # the padding behind the last token
            Z[m // 2, : e // 2] = -math.inf                # a column that half of the experts are closed to
        s["Z"] = Z.to(t)
        s["bias"] = 0.05 * normal(e) if case["bias"] else None
        s["scale"] = 2.5 if case["renorm"] else 1.0
        s["G"] = torch.empty(m, k, device="cuda")
        s["ir"] = torch.empty(m, k, dtype=torch.int32, device="cuda")
        s["jc"] = torch.empty(m + 1, dtype=torch.int32, device="cuda")
        s["counts"] = torch.empty(e, dtype=torch.int32, device="cuda")
        if op == "route_grad":
            w, ir, _, _ = _route(s)
            s["G"].copy_(w)
            s["ir"].copy_(ir)
            s["dG"] = normal(m, k)
            s["dZ"] = torch.empty(m, e, dtype=t, device="cuda")
    elif op in ("distill", "distill_grad"):
        v, m, k, t = case["v"], case["m"], case["k"], DTYPES[case["type"]]
        lengths = torch.full((m,), k, device="cuda")
        if case["ragged"]:
            lengths = torch.randint(1, k + 1, (m,), generator=g, device="cuda")
            if m > 4:
                lengths[m // 3] = 0                        # padding
                lengths[-1] = 0
        s["jc"], s["ic"] = _csc(lengths)
        s["ir"] = _distinct_rows(g, lengths, s["jc"], s["ic"], v)
        s["T"] = 3 + 2 * normal(s["ir"].numel())
        s["Z"] = torch.empty(m, v, dtype=t, device="cuda")
        for a in range(0, m, 512):
            s["Z"][a:a + 512] = (2 * normal(min(512, m - a), v)).to(t)
        # a mean over the columns; in half precision with the loss scale that keeps the gradient's values normal numbers
        s["weight"] = torch.rand(m, generator=g, device="cuda") * (1024.0 if case["type"] == "f16" else 1.0 / m)
        s["loss"] = torch.empty(m, device="cuda")
        s["lse"] = torch.empty(m, device="cuda")
        s["dZ"] = torch.empty(m, v, dtype=t, device="cuda")
        if op == "distill_grad":
            for a in range(0, m, 512):
                s["lse"][a:a + 512] = torch.logsumexp(s["Z"][a:a + 512].double() / case["tau"], 1).float()
    else:
        n, rows, cols = case["n"], case["rows"], case["cols"]
        if case["law"] == "pareto":
            u = torch.rand(cols, generator=g, device="cuda").clamp_min(1e-6)
            lengths = (case["mean"] / 3.0 * u ** (-1 / 1.5)).clamp(1, 50 * case["mean"]).long().clamp_max(rows)
        else:
            lengths = torch.full((cols,), min(case["mean"], rows), device="cuda")
        s["jc"], s["ic"] = _csc(lengths)
        nnz = s["ic"].numel()
        s["ir"] = torch.randint(0, rows, (nnz,), generator=g, device="cuda").int()
        s["S"] = 1 - torch.rand(nnz, generator=g, device="cuda")
        s["Q"] = torch.empty(rows, n, dtype=torch.float8_e4m3fn, device="cuda")
        for a in range(0, rows, 16384):
            s["Q"][a:a + 16384] = (100 * normal(min(16384, rows - a), n)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s["scales"] = 0.01 + 0.01 * torch.rand(rows, _ngroups(n, case["group"]), generator=g, device="cuda")
        s["C"] = torch.empty(cols, n, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms

def _norm(s):
    n, m = s["n"], s["m"]
    h = s["X"].float()
    if s["R"] is not None:
        h = h + s["R"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"]
    out = {}
    if s["H"] is not None:
        out["H"] = h.to(s["H"].dtype)
    if s["Y"] is not None:
        out["Y"] = y.to(s["Y"].dtype)
    if s["Q"] is not None:
        group = s["group"] or n
        ng = _ngroups(n, s["group"])
        padded = torch.nn.functional.pad(y, (0, ng * group - n)).view(m, ng, group)
        scales = (padded.abs().amax(2) / E4M3_MAX).clamp_min(SCALE_MIN)
        out["Q"] = (padded / scales[:, :, None]).view(m, ng * group)[:, :n].to(torch.float8_e4m3fn)
        out["scales"] = scales
    return out


def _norm_grad(s):
    h, g = s["H"].float(), s["dY"].float()
    rs = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    gw = g * s["w"]
    dx = rs * (gw - h * (rs * rs * (gw * h).mean(1, keepdim=True)))
    if s["dH"] is not None:
        dx = dx + s["dH"].float()
    return {"dX": dx.to(s["dX"].dtype), "dw": (g * h * rs).sum(0)}


def _scores(z, kind):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _route(s):
    z = s["Z"].double()
    m, e = z.shape
    p = _scores(z, s["kind"])
    key = z if s["bias"] is None and s["groups"] == 1 else p if s["bias"] is None else p + s["bias"].double()
    key = torch.where(z > -math.inf, key, -math.inf)
    if s["groups"] > 1:
        best = key.view(m, s["groups"], -1).sort(2, descending=True)[0][:, :, :2]
        total = torch.where(best > -math.inf, best, 0.0).sum(2)
        total = torch.where(best[:, :, 0] > -math.inf, total, -math.inf)
        taken = total.argsort(dim=1, descending=True, stable=True)[:, : s["topgroups"]]
        open_ = torch.zeros(m, s["groups"], dtype=torch.bool, device=z.device).scatter_(1, taken, True)
        key = torch.where(open_.repeat_interleave(e // s["groups"], 1), key, -math.inf)
    ir = key.argsort(dim=1, descending=True, stable=True)[:, : s["k"]].sort(1)[0]
    valid = key.gather(1, ir) > -math.inf
    w = torch.where(valid, p.gather(1, ir), 0.0)
    if s["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    counts = torch.bincount(ir.reshape(-1), weights=valid.reshape(-1).double(), minlength=e)
    jc = torch.arange(m + 1, device=z.device) * s["k"]
    return (w * s["scale"]).float(), ir.int(), jc.int(), counts.int()


def _route_grad(s):
    z, w, dg, ir = s["Z"].float(), s["G"], s["dG"], s["ir"].long()
    inner = (w * dg).sum(1, keepdim=True)
    if s["kind"] == "softmax" and not s["renorm"]:
        p = _scores(z, "softmax")
        up = torch.zeros_like(z).scatter_(1, ir, torch.where(w > 0, dg * s["scale"], 0.0))
        return (p * (up - inner)).to(s["dZ"].dtype)
    d = w * (dg - inner / s["scale"]) if s["renorm"] else w * dg
    if s["kind"] == "sigmoid":
        d = d / (1 + torch.exp(z.gather(1, ir)))
    d = torch.where(w > 0, d, 0.0)
    return torch.zeros_like(z).scatter_(1, ir, d).to(s["dZ"].dtype)


def _teacher(s):
    """p and log p of every entry, and which columns have entries."""
    m, ic = s["m"], s["ic"]
    t = s["T"] / s["tau"]
    top = torch.full((m,), -math.inf, device="cuda").scatter_reduce(0, ic, t, "amax")
    x = t - top[ic]
    total = torch.zeros(m, device="cuda").index_add(0, ic, torch.exp(x))
    logp = x - torch.log(total)[ic]
    return torch.exp(logp), logp, total > 0


def _distill(s, lse=None):
    ic, ir, tau = s["ic"], s["ir"].long(), s["tau"]
    x = s["Z"].float() / tau
    p, logp, some = _teacher(s)
    weight = torch.where(some, s["weight"], 0.0)
    out = {}
    if lse is None:
        top = x.amax(1)
        lse = top + torch.log(torch.exp(x - top[:, None]).sum(1))
        kl = torch.zeros(s["m"], device="cuda").index_add(0, ic, p * (logp - (x[ic, ir] - lse[ic])))
        out["loss"] = tau * tau * weight * kl
        out["lse"] = lse
    scale = weight * tau
    x = torch.exp(x.sub_(lse[:, None])).mul_(scale[:, None])
    x.index_put_((ic, ir), -p * scale[ic], accumulate=True)
    out["dZ"] = x.to(s["dZ"].dtype)
    return out


def _q8(s):
    n, ir = s["n"], s["ir"].long()
    group = s["group"] or n
    wide = (s["scales"][ir] * s["S"][:, None]).repeat_interleave(group, 1)[:, :n]
    wide = wide * s["Q"].view(torch.uint8)[ir].view(torch.float8_e4m3fn).float()
    return torch.zeros(s["cols"], n, device="cuda").index_add_(0, s["ic"], wide)


# ---------------------------------------------------------------- the library's calls

_abi = None


def _library():
    global _abi
    if _abi is None:
        from bidmat_amd import hip_abi
        _abi = hip_abi.load(), hip_abi.check
    return _abi


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    lib, check = _library()
    stream = torch.cuda.current_stream().cuda_stream
    op = s["op"]
    if op == "norm":
        n = s["n"]
        check(lib.bidmat_rmsnorm(n, s["m"], CODES[s["type"]], _p(s["X"]), n, _p(s["R"]), n, _p(s["w"]), EPS, _p(s["H"]), n, _p(s["Y"]), n,
                                 _p(s["Q"]), n, _p(s["scales"]), max(0, s["group"]), stream), "rmsnorm")
        return {k: s[k] for k in ("H", "Y", "Q", "scales") if s[k] is not None}
    if op == "norm_grad":
        n = s["n"]
        check(lib.bidmat_rmsnorm_grad(n, s["m"], CODES[s["type"]], _p(s["H"]), n, _p(s["w"]), EPS, _p(s["dY"]), n, _p(s["dH"]), n,
                                      _p(s["dX"]), n, _p(s["dw"]), 0, stream), "rmsnorm_grad")
        return {"dX": s["dX"], "dw": s["dw"]}
    if op == "route":
        check(lib.bidmat_route(s["e"], s["m"], CODES[s["type"]], _p(s["Z"]), s["e"], _p(s["bias"]), KINDS[s["kind"]], s["groups"],
                               s["topgroups"], s["k"], int(s["renorm"]), s["scale"], _p(s["G"]), _p(s["ir"]), None, _p(s["jc"]),
                               _p(s["counts"]), stream), "route")
        return {"G": s["G"], "ir": s["ir"], "jc": s["jc"], "counts": s["counts"]}
    if op == "route_grad":
        check(lib.bidmat_route_grad(s["e"], s["m"], CODES[s["type"]], _p(s["Z"]), s["e"], KINDS[s["kind"]], s["k"], int(s["renorm"]),
                                    s["scale"], _p(s["G"]), _p(s["ir"]), _p(s["dG"]), _p(s["dZ"]), s["e"], stream), "route_grad")
        return {"dZ": s["dZ"]}
    if op == "distill":
        v = s["v"]
        check(lib.bidmat_distill(v, s["m"], CODES[s["type"]], _p(s["Z"]), v, s["T"].numel(), _p(s["T"]), _p(s["ir"]), _p(s["jc"]),
                                 s["tau"], _p(s["weight"]), _p(s["loss"]), _p(s["lse"]), _p(s["dZ"]), v, stream), "distill")
        return {"loss": s["loss"], "lse": s["lse"], "dZ": s["dZ"]}
    if op == "distill_grad":
        v = s["v"]
        check(lib.bidmat_distill_grad(v, s["m"], CODES[s["type"]], _p(s["Z"]), v, s["T"].numel(), _p(s["T"]), _p(s["ir"]), _p(s["jc"]),
                                      s["tau"], _p(s["weight"]), _p(s["lse"]), _p(s["dZ"]), v, stream), "distill_grad")
        return {"dZ": s["dZ"]}
    check(lib.bidmat_dsmult_q8_csc(s["n"], s["cols"], s["S"].numel(), _p(s["Q"]), s["n"], _p(s["scales"]), s["group"], _p(s["S"]),
                                   _p(s["ir"]), _p(s["jc"]), _p(s["C"]), 0, stream), "dsmult_q8_csc")
    return {"C": s["C"]}


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "norm":
        return _norm(state)
    if op == "norm_grad":
        return _norm_grad(state)
    if op == "route":
        w, ir, jc, counts = _route(state)
        return {"G": w, "ir": ir, "jc": jc, "counts": counts}
    if op == "route_grad":
        return {"dZ": _route_grad(state)}
    if op == "distill":
        return _distill(state)
    if op == "distill_grad":
        return _distill(state, state["lse"])
    return {"C": _q8(state)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, m, b = case["n"], case["m"], DTYPES[case["type"]].itemsize
        if op == "norm":
            per = b * (1 + 2 * case["res"] + case["y"]) + (case["group"] >= 0)
            return {"bytes": per * n * m + 4 * n + (4 * m * _ngroups(n, case["group"]) if case["group"] >= 0 else 0), "flops": 6 * n * m}
        return {"bytes": b * (3 + case["res"]) * n * m + 8 * n, "flops": 10 * n * m}
    if op in ("route", "route_grad"):
        e, m, k, b = case["e"], case["m"], case["k"], DTYPES[case["type"]].itemsize
        if op == "route":
            return {"bytes": b * e * m + 8 * k * m + 4 * m + 4 * e * (1 + case["bias"]), "flops": 6 * e * m}
        reads = e if case["kind"] == "softmax" and not case["renorm"] else k if case["kind"] == "sigmoid" else 0
        return {"bytes": b * (e + reads) * m + 12 * k * m, "flops": 6 * e * m}
    if op in ("distill", "distill_grad"):
        v, m, b = case["v"], case["m"], DTYPES[case["type"]].itemsize
        entries = case["k"] * m / (2 if case["ragged"] else 1)
        return {"bytes": 2 * b * v * m + 8 * entries + 16 * m, "flops": 8 * v * m}
    nnz = case["cols"] * case["mean"]
    touched = case["rows"] * (1 - math.exp(-nnz / case["rows"]))    # columns of the table that some nonzero names
    return {"bytes": touched * (case["n"] + 4 * _ngroups(case["n"], case["group"])) + 8 * nnz + 4 * case["n"] * case["cols"],
            "flops": 2 * nnz * case["n"]}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_norm(s):
    h = s["X"].double()
    if s["R"] is not None:
        h += s["R"].double()
    out = {}
    if s["H"] is not None:
        out["H"] = h.clone()
    size = torch.linalg.vector_norm(h, dim=1) / math.sqrt(s["n"])
    h /= torch.sqrt(size ** 2 + EPS)[:, None]
    h *= s["w"].double()
    if s["Y"] is not None:
        out["Y"] = h.clone()
    if s["Q"] is not None:
        group = s["group"] or s["n"]
        scales = torch.stack([h[:, a:a + group].abs().amax(1) for a in range(0, s["n"], group)], 1) / E4M3_MAX
        scales = torch.maximum(scales, torch.tensor(SCALE_MIN, dtype=torch.float64, device=h.device))
        for i, a in enumerate(range(0, s["n"], group)):
            h[:, a:a + group] /= scales[:, i:i + 1]
        out["Q"], out["scales"] = h, scales
    return out


def _exact_norm_grad(s):
    n = s["n"]
    dx = torch.empty(s["m"], n, dtype=torch.float64, device="cuda")
    dw = torch.zeros(n, dtype=torch.float64, device="cuda")
    w = s["w"].double()
    for a in range(0, s["m"], 4096):
        h, g = s["H"][a:a + 4096].double(), s["dY"][a:a + 4096].double()
        size = torch.sqrt(torch.einsum("ij,ij->i", h, h) / n + EPS)[:, None]
        unit = h / size
        dw += (g * unit).sum(0)
        g *= w
        dx[a:a + 4096] = (g - unit * ((g * unit).sum(1, keepdim=True) / n)) / size
        if s["dH"] is not None:
            dx[a:a + 4096] += s["dH"][a:a + 4096].double()
    return {"dX": dx, "dw": dw}


def _exact_scores(z, kind):
    if kind == "sigmoid":
        return torch.sigmoid(z)
    return torch.softmax(z, 1).nan_to_num(0.0)


def _places(key):
    """How many entries of a column come before each: larger ones, and equal ones of a lower index."""
    before = key[:, None, :] > key[:, :, None]
    equal = key[:, None, :] == key[:, :, None]
    lower = torch.ones(key.shape[1], key.shape[1], dtype=torch.bool, device=key.device).tril(-1)
    return (before | (equal & lower)).sum(2)


def _exact_route(s):
    m, e, k, groups = s["m"], s["e"], s["k"], s["groups"]
    ws, irs, counts = [], [], torch.zeros(e, dtype=torch.int64, device="cuda")
    step = max(1, (1 << 27) // (e * e))
    for a in range(0, m, step):
        z = s["Z"][a:a + step].double()
        closed = torch.isinf(z) & (z < 0)
        p = _exact_scores(z, s["kind"])
        key = p.clone()
        if s["bias"] is not None:
            key += s["bias"].double()
        elif groups == 1:
            key = z.clone()
        key[closed] = -math.inf
        if groups > 1:
            parts = key.view(-1, e // groups)
            first = parts.amax(1)
            rest = parts.clone().scatter_(1, parts.argmax(1, keepdim=True), -math.inf).amax(1)
            total = torch.where(first == -math.inf, first, first + torch.where(rest == -math.inf, 0.0, rest)).view(-1, groups)
            key[(_places(total) >= s["topgroups"]).repeat_interleave(e // groups, 1)] = -math.inf
        taken = _places(key) < k
        ir = taken.nonzero()[:, 1].view(-1, k)
        valid = key.gather(1, ir) > -math.inf
        w = p.gather(1, ir) * valid
        if s["renorm"]:
            w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
        ws.append(w * s["scale"])
        irs.append(ir)
        counts += (taken & (key > -math.inf)).sum(0)
    return {"G": torch.cat(ws), "ir": torch.cat(irs).int(), "jc": torch.arange(0, m * k + 1, k, device="cuda").int(), "counts": counts.int()}


def _exact_route_grad(s):
    z, w, dg, ir = s["Z"].double(), s["G"].double(), s["dG"].double(), s["ir"].long()
    p = _exact_scores(z, s["kind"])
    chosen = torch.zeros_like(z).scatter_(1, ir, (w > 0).double())
    up = torch.zeros_like(z).scatter_(1, ir, dg) * chosen * s["scale"]
    if s["renorm"]:
        total = (p * chosen).sum(1, keepdim=True).clamp_min(1e-300)
        up = (up - (up * p * chosen).sum(1, keepdim=True) / total) / total * chosen
    if s["kind"] == "sigmoid":
        return {"dZ": up * p * torch.sigmoid(-z)}
    return {"dZ": p * (up - (up * p).sum(1, keepdim=True))}


def _exact_distill(s, with_loss):
    m, v, tau = s["m"], s["v"], s["tau"]
    loss, kept = torch.zeros(m, dtype=torch.float64, device="cuda"), torch.empty(m, dtype=torch.float64, device="cuda")
    grad = torch.empty(m, v, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // v)
    jc = s["jc"].tolist()
    for a in range(0, m, step):
        b = min(m, a + step)
        x = s["Z"][a:b].double() / tau
        lse = torch.logsumexp(x, 1) if with_loss else s["lse"][a:b].double()
        kept[a:b] = lse
        lo, hi = jc[a], jc[b]
        ic, ir = s["ic"][lo:hi] - a, s["ir"][lo:hi].long()
        longest = max(1, max(jc[i + 1] - jc[i] for i in range(a, b)))
        at = torch.arange(lo, hi, device="cuda") - s["jc"][a:b].long()[ic]
        t = torch.full((b - a, longest), -math.inf, dtype=torch.float64, device="cuda")
        t[ic, at] = s["T"][lo:hi].double() / tau
        logp = torch.log_softmax(t, 1)[ic, at]
        x -= lse[:, None]
        some = torch.zeros(b - a, dtype=torch.float64, device="cuda")
        some[ic] = 1.0
        weight = s["weight"][a:b].double() * some
        part = torch.zeros(b - a, dtype=torch.float64, device="cuda").index_add(0, ic, torch.exp(logp) * (logp - x[ic, ir]))
        loss[a:b] = part * weight * tau * tau
        x = torch.exp(x)
        x.index_put_((ic, ir), -torch.exp(logp), accumulate=True)
        grad[a:b] = x * (weight * tau)[:, None]
    return {"loss": loss, "lse": kept, "dZ": grad} if with_loss else {"dZ": grad}


def _exact_q8(s):
    n, cols = s["n"], s["cols"]
    group = s["group"] or n
    table = (s["Q"].float() * s["scales"].repeat_interleave(group, 1)[:, :n].double())
    out = torch.zeros(cols, n, dtype=torch.float64, device="cuda")
    for a in range(0, s["ir"].numel(), 1 << 18):
        part = slice(a, a + (1 << 18))
        out.index_add_(0, s["ic"][part], table[s["ir"][part].long()] * s["S"][part].double()[:, None])
    return {"C": out}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "norm_grad":
        return _exact_norm_grad(s)
    if op == "route":
        return _exact_route(s)
    if op == "route_grad":
        return _exact_route_grad(s)
    if op in ("distill", "distill_grad"):
        return _exact_distill(s, op == "distill")
    return _exact_q8(s)
