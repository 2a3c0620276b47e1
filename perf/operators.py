"""The network-block operators at the sizes they are used at: the gated feed-forward block and the norms around it.

`own = False` computes them from elementary torch operations in float32; `own = True` makes the calls a user makes
(roundtrip_amd.Engine: gated_ffn_dev, block_norm_dev and their backward passes).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
ALPHA = 0.2            # slope of the framework's leaky ReLU
RES, BRANCH = 0.9, 0.7  # scales of the residual and of the branch


def _ffn(name, T, d, f, dtype, act, train=False):
    return {"name": name, "op": "ffn", "T": T, "d": d, "f": f, "dtype": dtype, "act": act, "train": train}


def _norm(name, T, d, dtype, kind, rows_per_gate, train=False):
    return {"name": name, "op": "norm", "T": T, "d": d, "dtype": dtype, "kind": kind, "rows_per_gate": rows_per_gate,
            "train": train}


def listed():
    return [
        # one latent point through a small block of the framework's own widths: launch latency is what counts
        _ffn("ffn_one_small", 1, 512, 1024, "f32", "lrelu"),
        # one token of a large network: every weight is read once
        _ffn("ffn_one_large", 1, 4096, 16384, "bf16", "silu"),
        # a small serving batch
        _ffn("ffn_batch_24", 24, 4096, 8192, "bf16", "gelu"),
        # the 100 x 100 evaluation grid through a block in the framework's own type
        _ffn("ffn_grid_f32", 10000, 512, 1024, "f32", "lrelu"),
        # a long prompt
        _ffn("ffn_prompt", 8192, 4096, 16384, "bf16", "silu"),
        # a training step of a mid-sized network
        _ffn("ffn_train", 4096, 2048, 8192, "bf16", "silu", True),
        # a training step on a ragged batch with widths that no vector load divides
        _ffn("ffn_train_odd", 1777, 1001, 2731, "f16", "gelu", True),
        # norms of one token: latency
        _norm("norm_one", 1, 4096, "bf16", "rms", 0),
        # norms of a long prompt, one gate vector for each sequence
        _norm("norm_prompt", 16384, 4096, "bf16", "rms", 4096),
        # a training step in the framework's own type and width, one learnt scale vector for all rows
        _norm("norm_train_f32", 10000, 512, "f32", "layer", 10000, True),
        # a training step of a large network, ragged rows for a gate
        _norm("norm_train", 8191, 4096, "bf16", "rms", 1000, True),
        # the whole block in a row as it is served to a small batch: norm, feed-forward, norm with gate and residual
        {"name": "block_batch_8", "op": "block", "T": 8, "d": 2048, "f": 8192, "dtype": "bf16", "act": "silu",
         "kind": "rms", "rows_per_gate": 1, "train": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "norm", "block"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    step = rng.choice([1, 8, 64])
    T, d = _log(rng, 1, 16384), max(step, _log(rng, 16, 6000) // step * step)
    c = {"op": op, "T": T, "d": d, "dtype": dtype, "train": rng.random() < 0.4}
    if op != "norm":
        c["f"] = max(step, _log(rng, 32, 16384) // step * step)
        c["act"] = rng.choice(["silu", "gelu", "lrelu", "sigmoid"])
        most = 6.0 * 8192 * 4096 * 16384 / (30 if dtype == "f32" else 1) / (3 if c["train"] else 1)
        while 6.0 * c["T"] * d * c["f"] > most:
            c["T"] = c["T"] * 2 // 3
    if op != "ffn":
        c["kind"] = rng.choice(["rms", "layer"])
        c["rows_per_gate"] = rng.choice([0, 1, _log(rng, 1, c["T"]), c["T"]])
    return c


def work(case):
    e, T, d, train = SIZE[case["dtype"]], case["T"], case["d"], case["train"]
    b = f = 0
    if case["op"] != "norm":
        w = 3 * d * case["f"]
        f += 2 * T * w * (3 if train else 1)
        b += e * (w * (2 if train else 1))
    if case["op"] != "ffn":
        gates = -(-T // case["rows_per_gate"]) if case["rows_per_gate"] else 0
        b += e * (gates + 2) * d * (2 if train else 1)
        f += 12 * T * d * (3 if train else 1)
    # rows in and out: ffn x, out (dout, dx); norm x, branch, y, n (dy, dn, dx, dbranch); block x, y, n (dy, dn, dx)
    rows = {"ffn": (2, 4), "norm": (4, 8), "block": (3, 6)}[case["op"]][1 if train else 0]
    return {"bytes": b + e * rows * T * d, "flops": f}


def _inputs(case, seed):
    T, d, dtype = case["T"], case["d"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    s = {"x": normal((T, d))}
    if case["op"] != "norm":
        f = case["f"]
        s["w_gate"], s["w_up"] = normal((d, f), d ** -0.5), normal((d, f), d ** -0.5)
        s["w_down"] = normal((f, d), f ** -0.5)
        if case["op"] == "ffn" and case["train"]:
            s["dout"] = normal((T, d))
    if case["op"] != "ffn":
        r = case["rows_per_gate"]
        s["w_post"], s["w_pre"] = normal((d,), 0.1, 1.0), normal((d,), 0.1, 1.0)
        s["gate"] = normal((-(-T // r), d), 0.5) if r else None
        if case["op"] == "norm":
            s["branch"] = normal((T, d), 1.5, 0.1)
        else:
            s["w_in"] = normal((d,), 0.1, 1.0)
        if case["train"]:
            s["dy"], s["dn"] = normal((T, d)), normal((T, d))
    return s


_engines = {}


def _engine():
    from roundtrip_amd import Engine
    dev = torch.cuda.current_device()
    if dev not in _engines:
        _engines[dev] = Engine(dev)
    return _engines[dev]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    # what a program keeps: the engine, its output and workspace buffers, and the description of the call
    eng = s["eng"] = _engine()
    T, d, dtype, train = case["T"], case["d"], DTYPES[case["dtype"]], case["train"]
    code = {"f32": eng.F32, "bf16": eng.BF16, "f16": eng.F16}[case["dtype"]]

    def new(*shape):
        return torch.empty(shape, dtype=dtype, device="cuda")

    out, p = {}, (lambda t: None if t is None else t.data_ptr())
    ws = 0
    if case["op"] != "norm":
        f = case["f"]
        act = {"silu": eng.SILU, "gelu": eng.GELU_TANH, "lrelu": eng.LRELU, "sigmoid": eng.SIGMOID}[case["act"]]
        x = s["x"] if case["op"] == "ffn" else new(T, d)
        b = new(T, d)
        s["pre"] = [torch.empty((T, f), device="cuda") if train else None for _ in range(2)]       # float32 in every type
        # the norm before hands over what its rounding left off too: the sign of a gate hangs on it
        lo = s["lo"] = new(T, d) if case["op"] == "block" and case["dtype"] != "f32" else None
        s["ffn"] = eng.gated_ffn_args(T, d, f, d, code, act, x=p(x), x_lo=p(lo), w_gate=p(s["w_gate"]), w_up=p(s["w_up"]),
                                      w_down=p(s["w_down"]), out=p(b), pre_gate=p(s["pre"][0]), pre_up=p(s["pre"][1]),
                                      alpha=ALPHA)
        ws = eng.gated_ffn_workspace(s["ffn"])
        if train:
            dx, wg, wu, wd = new(T, d), new(d, f), new(d, f), new(f, d)
            out.update(dw_gate=wg, dw_up=wu, dw_down=wd)
            dout = s["dout"] if case["op"] == "ffn" else new(T, d)
            s["ffn_grads"] = eng.gated_ffn_grads(dout=p(dout), dx=p(dx), dw_gate=p(wg), dw_up=p(wu), dw_down=p(wd))
            ws = max(ws, eng.gated_ffn_workspace(s["ffn"], backward=True))
            s["keep"] = (dout, dx)
        if case["op"] == "ffn":
            out["out"] = b
            if train:
                out["dx"] = dx
        else:
            s["hidden"] = (x, b)
    if case["op"] != "ffn":
        kind = {"rms": eng.RMS, "layer": eng.LAYER}[case["kind"]]
        branch = s["branch"] if case["op"] == "norm" else b
        y, n = out["y"], out["n"] = new(T, d), new(T, d)
        s["norm"] = eng.block_norm_args(T, d, code, kind, x=p(s["x"]), branch=p(branch), y=p(y), n=p(n),
                                        w_post=p(s["w_post"]), w_pre=p(s["w_pre"]), gate=p(s["gate"]),
                                        rows_per_gate=case["rows_per_gate"] or 1, res_scale=RES, branch_scale=BRANCH,
                                        eps=EPS)
        if train:
            dx = out["dx"] = new(T, d)
            db = new(T, d) if case["op"] == "norm" else dout
            if case["op"] == "norm":
                out["dbranch"] = db
            out["dw_post"], out["dw_pre"] = new(d), new(d)
            out["dgate"] = None if s["gate"] is None else torch.empty_like(s["gate"])
            s["norm_grads"] = eng.block_norm_grads(dy=p(s["dy"]), dn=p(s["dn"]), dx=p(dx), dbranch=p(db),
                                                   dgate=p(out["dgate"]), dw_post=p(out["dw_post"]),
                                                   dw_pre=p(out["dw_pre"]))
            ws = max(ws, eng.block_norm_workspace(s["norm"]))
        if case["op"] == "block":
            # the norm before: of the block's input, with no branch; its gradient joins the residual's
            s["norm_in"] = eng.block_norm_args(T, d, code, kind, x=p(s["x"]), n=p(x), n_lo=p(lo), w_pre=p(s["w_in"]), eps=EPS)
            if train:
                out["dw_in"] = new(d)
                s["norm_in_grads"] = eng.block_norm_grads(dy=p(dx), dn=p(s["keep"][1]), dx=p(dx),
                                                          dw_pre=p(out["dw_in"]))
                ws = max(ws, eng.block_norm_workspace(s["norm_in"]))
    s["ws"] = torch.empty(max(ws, 1), dtype=torch.uint8, device="cuda")
    s["out"] = out
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


class _Held(object):
    """Goes with its state, and waits then for the passes that use the state's arrays."""

    def __init__(self, eng):
        self.eng = eng

    def __del__(self):
        self.eng.sync()


def _join_streams(s):
    """The calls run on the engine's stream and the arrays are torch's; neither stream waits for the other by itself.  From a
    state's first pass on: its inputs are there, and no array goes to another owner while a pass uses it.  Outputs are read when
    the device, or the engine (`Engine.sync`), has been waited for."""
    torch.cuda.ExternalStream(s["eng"].stream).wait_stream(torch.cuda.current_stream())
    s["held"] = _Held(s["eng"])


def _run_own(s):
    eng, case = s["eng"], s["case"]
    if "held" not in s:
        _join_streams(s)
    ws, size = s["ws"].data_ptr(), s["ws"].numel()
    if case["op"] == "block":
        eng.block_norm_dev(s["norm_in"])
    if case["op"] != "norm":
        eng.gated_ffn_dev(s["ffn"], ws, size)
    if case["op"] != "ffn":
        eng.block_norm_dev(s["norm"])
    if case["train"]:
        if case["op"] != "ffn":
            eng.block_norm_backward_dev(s["norm"], s["norm_grads"], ws, size)
        if case["op"] != "norm":
            eng.gated_ffn_backward_dev(s["ffn"], s["ffn_grads"], ws, size)
        if case["op"] == "block":
            eng.block_norm_backward_dev(s["norm_in"], s["norm_in_grads"], ws, size)
    return s["out"]


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _act(kind, g):
    """act(g) and its derivative."""
    if kind == "lrelu":
        one = torch.where(g > 0, 1.0, ALPHA)
        return g * one, one
    if kind == "gelu":
        c = math.sqrt(2.0 / math.pi)
        t = 1.0 - 2.0 / (torch.exp(2.0 * c * (g + 0.044715 * g * g * g)) + 1.0)
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)
    sg = 1.0 / (1.0 + torch.exp(-g))
    if kind == "sigmoid":
        return sg, sg * (1.0 - sg)
    return g * sg, sg * (1.0 + g * (1.0 - sg))


def _ffn_plain(act, x, wg, wu, wd):
    g, u = x @ wg, x @ wu
    a, da = _act(act, g)
    h = a * u
    return h @ wd, (x, wg, wu, wd, u, a, da, h)


def _ffn_back_plain(kept, dout):
    x, wg, wu, wd, u, a, da, h = kept
    dh = dout @ wd.t()
    dg, du = dh * u * da, dh * a
    return dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du, h.t() @ dout


def _hat(kind, v):
    """The normed rows before their weight, and the factor of each row."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    return v * r, r


def _hat_back(kind, vh, r, z):
    z = z - vh * (z * vh).mean(1, keepdim=True)
    if kind == "layer":
        z = z - z.mean(1, keepdim=True)
    return z * r


def _rows_of_gate(gate, r, T):
    return gate[torch.arange(T, device=gate.device) // r]


def _run_plain(s):
    case = s["case"]
    T, dtype = case["T"], DTYPES[case["dtype"]]
    v = {k: t.float() for k, t in s.items() if isinstance(t, torch.Tensor)}
    out, x = {}, v["x"]
    if case["op"] == "ffn":
        out["out"], kept = _ffn_plain(case["act"], x, v["w_gate"], v["w_up"], v["w_down"])
        if case["train"]:
            out["dx"], out["dw_gate"], out["dw_up"], out["dw_down"] = _ffn_back_plain(kept, v["dout"])
        return {k: t.to(dtype) for k, t in out.items()}
    kind, r = case["kind"], case["rows_per_gate"]
    if case["op"] == "block":
        xh, xr = _hat(kind, x)
        b, kept = _ffn_plain(case["act"], xh * v["w_in"], v["w_gate"], v["w_up"], v["w_down"])
    else:
        b = v["branch"]
    bh, br = _hat(kind, b)
    gate = _rows_of_gate(v["gate"], r, T) if r else 1.0
    out["y"] = RES * x + BRANCH * gate * (bh * v["w_post"])
    yh, yr = _hat(kind, out["y"])
    out["n"] = yh * v["w_pre"]
    if case["train"]:
        t = v["dy"] + _hat_back(kind, yh, yr, v["dn"] * v["w_pre"])
        q = BRANCH * gate * t
        db = _hat_back(kind, bh, br, q * v["w_post"])
        out["dw_post"], out["dw_pre"] = (q * bh).sum(0), (v["dn"] * yh).sum(0)
        if r:
            q = torch.zeros((v["gate"].shape[0] * r, case["d"]), device=x.device)
            q[:T] = BRANCH * t * (bh * v["w_post"])
            out["dgate"] = q.view(-1, r, case["d"]).sum(1)
        dx = RES * t
        if case["op"] == "block":
            dn, out["dw_gate"], out["dw_up"], out["dw_down"] = _ffn_back_plain(kept, db)
            out["dw_in"] = (dn * xh).sum(0)
            dx = dx + _hat_back(kind, xh, xr, dn * v["w_in"])
        else:
            out["dbranch"] = db
        out["dx"] = dx
    return {k: t.to(dtype) for k, t in out.items()}


# ---- the definition in 64 bits: values by the formulas' own torch functions, gradients by differentiation --------
def exact(case, seed):
    s = {k: t.double() for k, t in _inputs(case, seed).items() if t is not None}
    T, d, train = case["T"], case["d"], case["train"]
    names = [k for k in s if k not in ("dout", "dy", "dn")] if train else []
    for k in names:
        s[k].requires_grad_(True)

    def norm(v, w):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(v, (d,), w, None, EPS)
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + EPS) * w

    def ffn(v):
        a = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid,
             "gelu": lambda g: torch.nn.functional.gelu(g, approximate="tanh"),
             "lrelu": lambda g: torch.nn.functional.leaky_relu(g, ALPHA)}[case["act"]]
        return torch.mm(a(torch.mm(v, s["w_gate"])) * torch.mm(v, s["w_up"]), s["w_down"])

    with torch.set_grad_enabled(train):
        if case["op"] == "ffn":
            out, seeds = {"out": ffn(s["x"])}, ["dout"]
        else:
            b = s["branch"] if case["op"] == "norm" else ffn(norm(s["x"], s["w_in"]))
            b = norm(b, s["w_post"]) * BRANCH
            if case["rows_per_gate"]:
                b = b * s["gate"].repeat_interleave(case["rows_per_gate"], 0)[:T]
            y = s["x"] * RES + b
            out, seeds = {"y": y, "n": norm(y, s["w_pre"])}, ["dy", "dn"]
        if train:
            got = torch.autograd.grad(list(out.values()), [s[k] for k in names], [s[k] for k in seeds])
            out.update(("d" + k, g) for k, g in zip(names, got))
    return {k: t.detach() for k, t in out.items()}
