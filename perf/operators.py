"""The feed-forward sublayer's operators, as cases that can be timed.

  norm            layer norm over the last axis (Context.layer_norm)
  norm_backward   its gradients: dx, and dw and db summed over the rows
                  (Context.layer_norm_backward)
  gated           silu(x Wg^T) * (x Wu^T) (Context.gated_contract_bf16)
  gated_backward  its gradients: dx, dWg, dWu
                  (Context.gated_contract_bf16_backward)
  linear_i8       rows quantized to 8 bits with a scale each, then the product
                  with weights held in 8 bits with a scale for each channel
                  (Context.quantize_rows_i8, Context.contract_i8)

With `own` false a case runs in plain torch operations; with `own` true
through the public entry points of `tiler_amd`.  Device storage is torch's;
the framework's launches go to the bound context's stream.
"""
import math

import torch

own = False

EPS_BITS = 0x3727C5AC  # 1e-5 as binary32
EPS = 9.999999747378752e-06

_context = _workspace = None


def context():
    """The program's one bound context."""
    global _context
    if _context is None:
        from tiler_amd import Context
        _context = Context(0)
    return _context


def workspace(nbytes):
    """The program's one workspace, as large as its calls have needed so far (they follow one another on one stream)."""
    global _workspace
    if _workspace is None or _workspace.numel() < nbytes:
        context().synchronize()  # nothing reads the smaller one any more
        _workspace = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return _workspace


def listed():
    return [
        # A decode step's normalization: a token of each of 16 sequences.
        {"name": "norm_decode", "kind": "norm", "rows": 16, "extent": 4096, "dtype": "bf16", "train": False},
        # A training step's hidden states; mean and reciprocal deviation kept for the gradients.
        {"name": "norm_train", "kind": "norm", "rows": 8192, "extent": 4096, "dtype": "bf16", "train": True},
        # The gradients of the same.
        {"name": "norm_grad", "kind": "norm_backward", "rows": 8192, "extent": 4096, "dtype": "bf16"},
        # A small model in binary32, its width and its tokens ragged.
        {"name": "norm_grad_ragged", "kind": "norm_backward", "rows": 1237, "extent": 1023, "dtype": "f32"},
        # One token of each of 16 sequences: the weights' bytes.
        {"name": "gated_decode", "kind": "gated", "m": 16, "n": 14336, "k": 4096, "train": False},
        # A chunk of a prompt, an odd number of tokens.
        {"name": "gated_chunk", "kind": "gated", "m": 301, "n": 14336, "k": 4096, "train": False},
        # A training step, both projections kept for the gradients.
        {"name": "gated_train", "kind": "gated", "m": 4096, "n": 14336, "k": 4096, "train": True},
        # The gradients of the same.
        {"name": "gated_grad", "kind": "gated_backward", "m": 4096, "n": 14336, "k": 4096},
        # A small model whose widths and tokens are all odd.
        {"name": "gated_grad_ragged", "kind": "gated_backward", "m": 777, "n": 1365, "k": 509},
        # An 8-bit projection for one token of each of 16 sequences.
        {"name": "linear_i8_decode", "kind": "linear_i8", "m": 16, "n": 4096, "k": 4096, "out": "bf16"},
        # The same projection for a prompt.
        {"name": "linear_i8_prefill", "kind": "linear_i8", "m": 4096, "n": 4096, "k": 4096, "out": "bf16"},
        # Logits of a ragged batch: every extent odd, binary32 out.
        {"name": "linear_i8_ragged", "kind": "linear_i8", "m": 257, "n": 5001, "k": 1111, "out": "f32"},
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm_backward", "gated", "gated", "gated_backward", "linear_i8", "linear_i8"))
    if kind in ("norm", "norm_backward"):
        extent = rng.choice((512, 1024, 4096, 8192, _log(rng, 60, 20000), _log(rng, 60, 20000)))
        case = {"kind": kind, "rows": _log(rng, 1, min(8192, (1 << 25) // extent)), "extent": extent,
                "dtype": rng.choice(("bf16", "bf16", "f32"))}
        if kind == "norm":
            case["train"] = rng.random() < 0.5
        return case

    def width(hi):
        return rng.choice((1024, 2048, 4096, 8 * _log(rng, 32, hi // 8), _log(rng, 200, hi)))

    if kind == "linear_i8":
        return {"kind": kind, "m": _log(rng, 1, 4096), "n": width(14336), "k": width(8192),
                "out": rng.choice(("bf16", "bf16", "f32"))}
    case = {"kind": kind, "m": _log(rng, 1, 4096), "n": width(14336), "k": width(4096)}
    if kind == "gated":
        case["train"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# Inputs

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _normal(g, shape, std=1.0, dtype=torch.bfloat16, mean=0.0):
    """Seeded normal values (made in binary32, then narrowed)."""
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _quantize(x):
    """Rows in 8 bits: the scale in binary32, and the codes by the exact
    quotient to the nearest, ties to even (quotients in 64 bits: values next
    to a tie, and a scale of one step less gives other codes)."""
    scale = (x.abs().amax(-1).double() / 127.0).float().clamp_min(2.0 ** -126)
    return torch.round(x.double() / scale.double()[:, None]), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def new(dtype, *shape):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind in ("norm", "norm_backward"):
        rows, extent, dtype = case["rows"], case["extent"], _DTYPES[case["dtype"]]
        # hidden states with an offset and a spread of their own in each row
        x = _normal(g, (rows, extent), dtype=torch.float32)
        x = x * torch.rand((rows, 1), generator=g, device="cuda").add_(0.5) + _normal(g, (rows, 1), 0.5, torch.float32)
        s = {"x": x.to(dtype), "w": _normal(g, (extent,), 0.1, dtype, 1.0)}
        s["y"] = new(dtype, rows, extent)
        if kind == "norm":
            s["b"] = _normal(g, (extent,), 0.1, dtype)
            if case["train"]:
                s["mean"], s["rstd"] = new(torch.float32, rows), new(torch.float32, rows)
        else:
            s["dy"] = _normal(g, (rows, extent), 0.02, dtype)
            # what the forward pass kept
            wide = s["x"].double()
            s["mean"] = wide.mean(-1).float()
            s["rstd"] = (wide.var(-1, unbiased=False) + EPS).rsqrt().float()
            s["dw"], s["db"] = new(dtype, extent), new(dtype, extent)
    elif kind in ("gated", "gated_backward"):
        m, n, k = case["m"], case["n"], case["k"]
        s = {"x": _normal(g, (m, k)), "wg": _normal(g, (n, k), k ** -0.5), "wu": _normal(g, (n, k), k ** -0.5)}
        if kind == "gated":
            s["h"] = new(torch.bfloat16, m, n)
            if case["train"]:
                s["gate"], s["up"] = new(torch.bfloat16, m, n), new(torch.bfloat16, m, n)
        else:
            # what the forward pass kept
            s["gate"] = (s["x"].float() @ s["wg"].float().T).bfloat16()
            s["up"] = (s["x"].float() @ s["wu"].float().T).bfloat16()
            s["dh"] = _normal(g, (m, n), 0.02)
            s["dx"], s["dwg"], s["dwu"] = (new(torch.bfloat16, m, k), new(torch.bfloat16, n, k),
                                           new(torch.bfloat16, n, k))
    else:
        m, n, k = case["m"], case["n"], case["k"]
        # activations whose columns differ in size, as hidden states' do
        x = _normal(g, (m, k), dtype=torch.float32) * torch.exp(_normal(g, (k,), 0.5, torch.float32))
        codes, scale = _quantize(_normal(g, (n, k), k ** -0.5))
        s = {"x": x.bfloat16(), "weight": codes.to(torch.int8), "weight_scale": scale}
        s["q"], s["scale"] = new(torch.int8, m, k), new(torch.float32, m)
        s["c"] = new(_DTYPES[case["out"]], m, n)
    s["case"] = case
    return s


def _code(dtype):
    from tiler_amd import _lib as L
    return {"bf16": L.BF16, "f32": L.F32}[dtype]


# ---------------------------------------------------------------------------
# One pass

def _run_own(s):
    from tiler_amd import _lib as L
    case, ctx = s["case"], context()
    at = {name: v.data_ptr() for name, v in s.items() if isinstance(v, torch.Tensor)}
    kind = case["kind"]
    if kind == "norm":
        ctx.layer_norm(_code(case["dtype"]), at["x"], at["w"], at["b"], case["rows"], case["extent"], EPS_BITS,
                       at["y"], mean=at.get("mean"), rstd=at.get("rstd"))
        return {name: s[name] for name in ("y", "mean", "rstd") if name in s}
    if kind == "norm_backward":
        dtype = _code(case["dtype"])
        space = workspace(ctx.layer_norm_backward_workspace(dtype, case["rows"], case["extent"]))
        ctx.layer_norm_backward(dtype, at["dy"], at["x"], at["w"], at["mean"], at["rstd"], case["rows"],
                                case["extent"], at["y"], at["dw"], at["db"], workspace=space.data_ptr(),
                                workspace_bytes=space.numel())
        return {"dx": s["y"], "dw": s["dw"], "db": s["db"]}
    if kind == "gated":
        ctx.gated_contract_bf16(at["x"], at["wg"], at["wu"], case["m"], case["n"], case["k"], at["h"],
                                gate=at.get("gate"), up=at.get("up"))
        return {name: s[name] for name in ("h", "gate", "up") if name in s}
    if kind == "gated_backward":
        space = workspace(ctx.gated_contract_bf16_backward_workspace(case["m"], case["n"], case["k"]))
        ctx.gated_contract_bf16_backward(at["x"], at["wg"], at["wu"], at["gate"], at["up"], at["dh"], case["m"],
                                         case["n"], case["k"], at["dx"], at["dwg"], at["dwu"],
                                         workspace=space.data_ptr(), workspace_bytes=space.numel())
        return {"dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"]}
    ctx.quantize_rows_i8(L.BF16, at["x"], case["m"], case["k"], at["q"], at["scale"])
    ctx.contract_i8(at["q"], at["weight"], at["scale"], at["weight_scale"], case["m"], case["n"], case["k"],
                    _code(case["out"]), at["c"])
    return {"c": s["c"], "scale": s["scale"]}


def run(s):
    if own:
        return _run_own(s)
    case, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        x = s["x"].float()
        mean = x.mean(-1, keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
        out = {"y": (d * rstd * s["w"].float() + s["b"].float()).to(s["x"].dtype)}
        if case["train"]:
            out.update(mean=mean[:, 0], rstd=rstd[:, 0])
        return out
    if kind == "norm_backward":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xh = (s["x"].float() - s["mean"][:, None]) * rstd
        g = dy * s["w"].float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        dtype = s["x"].dtype
        return {"dx": dx.to(dtype), "dw": (dy * xh).sum(0).to(dtype), "db": dy.sum(0).to(dtype)}
    if kind == "gated":
        x = s["x"].float()
        gate, up = x @ s["wg"].float().T, x @ s["wu"].float().T
        out = {"h": (gate / (1.0 + torch.exp(-gate)) * up).bfloat16()}
        if case["train"]:
            out.update(gate=gate.bfloat16(), up=up.bfloat16())
        return out
    if kind == "gated_backward":
        x, gate, up, dh = (s[name].float() for name in ("x", "gate", "up", "dh"))
        sig = 1.0 / (1.0 + torch.exp(-gate))
        dgate, dup = dh * up * sig * (1.0 + gate * (1.0 - sig)), dh * gate * sig
        return {"dx": (dgate @ s["wg"].float() + dup @ s["wu"].float()).bfloat16(),
                "dwg": (dgate.T @ x).bfloat16(), "dwu": (dup.T @ x).bfloat16()}
    codes, scale = _quantize(s["x"])
    # in 64 bits: binary32 loses the integer sum beyond 2^24
    total = (codes @ s["weight"].double().T).float()
    return {"c": (total * scale[:, None] * s["weight_scale"]).to(s["c"].dtype), "scale": scale}


# ---------------------------------------------------------------------------
# What a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        n, e = case["rows"] * case["extent"], 2 if case["dtype"] == "bf16" else 4
        if kind == "norm":
            return {"bytes": 2 * n * e + 2 * case["extent"] * e + (8 * case["rows"] if case["train"] else 0),
                    "flops": 8 * n}
        return {"bytes": 3 * n * e + 3 * case["extent"] * e + 8 * case["rows"], "flops": 14 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "gated":
        return {"bytes": 2 * (m * k + 2 * n * k + (3 if case["train"] else 1) * m * n), "flops": 4 * m * n * k}
    if kind == "gated_backward":
        return {"bytes": 2 * (2 * m * k + 4 * n * k + 3 * m * n), "flops": 8 * m * n * k}
    out = 2 if case["out"] == "bf16" else 4
    return {"bytes": 2 * m * k + n * k + 4 * n + 4 * m + out * m * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# The same results from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    d = {name: v.double() for name, v in s.items() if isinstance(v, torch.Tensor)}
    if kind == "norm":
        var, mean = torch.var_mean(d["x"], -1, correction=0)
        rstd = (var + EPS) ** -0.5
        out = {"y": torch.addcmul(d["b"], (d["x"] - mean[:, None]) * rstd[:, None], d["w"])}
        if case["train"]:
            out.update(mean=mean, rstd=rstd)
        return out
    if kind == "norm_backward":
        # dx is r (I - 1 1^T / N - xh xh^T / N) (w * dy), the Jacobian's rows
        xh = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None]
        g = d["w"] * d["dy"]
        n = case["extent"]
        dx = g - g.sum(-1, keepdim=True) / n
        dx -= xh * (torch.linalg.vecdot(g, xh)[:, None] / n)
        return {"dx": dx * d["rstd"][:, None], "dw": torch.linalg.vecdot(d["dy"], xh, dim=0), "db": d["dy"].sum(0)}
    if kind == "gated":
        gate, up = torch.mm(d["x"], d["wg"].t()), torch.mm(d["x"], d["wu"].t())
        out = {"h": gate * torch.sigmoid(gate) * up}
        if case["train"]:
            out.update(gate=gate, up=up)
        return out
    if kind == "gated_backward":
        sig = torch.sigmoid(d["gate"])
        silu = d["gate"] * sig
        dup, dgate = d["dh"] * silu, d["dh"] * d["up"] * (sig + silu - silu * sig)
        return {"dx": torch.mm(dgate, d["wg"]) + torch.mm(dup, d["wu"]), "dwg": torch.mm(dgate.t(), d["x"]),
                "dwu": torch.mm(dup.t(), d["x"])}
    # the scale is a binary32 number of the operator, the codes whole numbers
    largest = torch.linalg.vector_norm(d["x"], float("inf"), dim=-1)
    scale = torch.clamp((largest / 127).float(), min=2.0 ** -126).double()
    codes = (d["x"] / scale.unsqueeze(-1)).round()
    return {"c": torch.mm(codes, d["weight"].t()) * torch.outer(scale, d["weight_scale"]), "scale": scale}
