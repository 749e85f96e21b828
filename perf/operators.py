"""Sequence operators as a language model's token mixer uses them, at the sizes that this package is used at.

* ``cs2d.gated_scan_1d``: the gated linear recurrence ``h[t] = a[t] * h[t-1] + b[t]`` over the tokens of a batch
  ``(batch, length, dim)`` or of packed sequences ``(total, dim)``, with the gradients of its inputs;
* ``cs2d.gated_scan_step``: one token of it, on a state that stays in place;
* ``cs2d.layer_norm``: layer normalisation with an optional SiLU gate behind it, of tokens or of the channel-major
  images that the scans write, with the gradients of its inputs and parameters.

Widths are the channel counts of ``cs2d.synthetic.CONFIGS`` (192 to 1536), lengths the numbers of pixels of its
feature maps (7x7 to 200x336) or generic.  A training case is the forward and every gradient in one pass, an
evaluation case the forward alone.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5
_MOST = 1 << 27          # elements of one activation tensor of the largest case


def _scan(name, mode, dtype, form, weighted, batch, length, dim, seqs=0, h0=True):
    return {"name": name, "op": "scan", "mode": mode, "dtype": dtype, "form": form, "weighted": weighted, "batch": batch,
            "length": length, "dim": dim, "seqs": seqs, "h0": h0}


def _norm(name, mode, dtype, layout, gated, batch, h, w, dim):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "layout": layout, "gated": gated, "batch": batch, "h": h,
            "w": w, "dim": dim}


def listed():
    return [
        # one token of one request: a launch and the host's work
        _scan("step_one_bf16", "step", "bf16", "sigmoid", True, 1, 1, 384),
        # one token of a full serving batch
        _scan("step_batch_fp16", "step", "fp16", "log", True, 512, 1, 1536),
        # a prompt of one request: few channels, the length of a 56x56 map
        _scan("prompt_eval_bf16", "eval", "bf16", "sigmoid", True, 1, 3136, 192),
        # an ordinary training batch
        _scan("train_bf16", "train", "bf16", "sigmoid", True, 8, 4096, 768, h0=False),
        # one long sequence (a 200x336 map in reading order), trained in pieces: the state comes in and its gradient goes out
        _scan("long_train_bf16", "train", "bf16", "log", False, 1, 67200, 384),
        # documents of all lengths packed into one batch, some of them empty, padding behind the last one; nothing divides anything
        _scan("packed_train_fp32", "train", "fp32", "sigmoid", True, 1, 25111, 387, seqs=61),
        # the largest: gates that the caller computed
        _scan("large_train_bf16", "train", "bf16", "direct", False, 16, 16384, 512, h0=False),
        # the last stage of one image: few rows, wide ones
        _norm("few_rows_eval_fp32", "eval", "fp32", "tokens", False, 1, 7, 7, 1536),
        # first-stage tokens of a training batch
        _norm("tokens_train_bf16", "train", "bf16", "tokens", False, 32, 56, 56, 192),
        # third-stage tokens in full precision, with the gate of the block
        _norm("gated_train_fp32", "train", "fp32", "tokens", True, 128, 14, 14, 768),
        # what the four-corner operator writes for a segmentation map, normalised over its channels and gated
        _norm("image_gated_train_bf16", "train", "bf16", "image", True, 16, 128, 128, 384),
        # nothing divides anything: odd rows, an odd number of channels, half precision
        _norm("ragged_image_train_fp16", "train", "fp16", "image", True, 3, 45, 61, 51),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    dim = rng.choice([192, 384, 768, 1536, _log(rng, 8, 1536), _log(rng, 8, 1536)])
    most = _MOST // 2 if dtype == "fp32" else _MOST
    if rng.random() < 0.55:
        mode = rng.choice(["step", "eval", "train", "train"])
        form, weighted, h0 = rng.choice(["sigmoid", "log", "direct"]), rng.random() < 0.5, rng.random() < 0.6
        if mode == "step":
            return _unnamed(_scan("", mode, dtype, form, weighted, _log(rng, 1, 1024), 1, dim))
        length = _log(rng, 1, 67200)
        if rng.random() < 0.3:
            seqs = min(512, _log(rng, 1, max(2, length // 4)))
            return _unnamed(_scan("", mode, dtype, form, weighted, 1, min(length, most // dim), dim, seqs, h0))
        batch = max(1, min(_log(rng, 1, 128), most // (length * dim)))
        return _unnamed(_scan("", mode, dtype, form, weighted, batch, min(length, most // dim), dim, 0, h0))
    h = _log(rng, 1, 200)
    w = max(1, int(round(h * rng.uniform(0.6, 1.7))))
    batch = max(1, min(_log(rng, 1, 128), most // (h * w * dim)))
    return _unnamed(_norm("", rng.choice(["eval", "train", "train"]), dtype, rng.choice(["tokens", "image"]), rng.random() < 0.6,
                          batch, h, w, dim))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _offsets(gen, total, seqs, dev):
    """Borders of `seqs` sequences of all lengths: some empty, a few rows behind the last one."""
    used = total - total // 50
    cuts = (torch.rand(seqs - 1, generator=gen, device=dev) * (used + 1)).long().clamp(max=used).sort().values
    if seqs > 4:
        cuts[seqs // 2] = cuts[seqs // 2 - 1]
    ends = torch.tensor([0, used], device=dev)
    return torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)


def prepare(case, seed):
    dev, dtype = "cuda", _DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    train = case["mode"] == "train"

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        b, h, w, d = (case[k] for k in ("batch", "h", "w", "dim"))
        shape = (b, d, h, w) if case["layout"] == "image" else (b, h, w, d)
        per_channel = (1, d, 1, 1) if case["layout"] == "image" else (d,)
        s["x"] = (randn(*shape) * (0.5 + torch.rand(d, generator=gen, device=dev)).view(per_channel) + randn(d).view(per_channel)).to(dtype)
        s["weight"], s["bias"] = 1.0 + 0.1 * randn(d), 0.1 * randn(d)
        s["gate"] = randn(b, h, w, d).to(dtype) if case["gated"] else None
        leaves = ["x", "weight", "bias", "gate"]
        if train:
            s["dy"] = randn(b, h, w, d).to(dtype)
    else:
        b, n, d = (case[k] for k in ("batch", "length", "dim"))
        shape = (n, d) if case["seqs"] else (b, d) if case["mode"] == "step" else (b, n, d)
        states = case["seqs"] or b
        s["u"] = randn(*shape).to(dtype)
        # gates that keep for a few to a few thousand tokens
        if case["form"] == "sigmoid":
            gate = 3.0 + 2.0 * randn(*shape)
        else:
            gate = -torch.exp(1.5 * randn(*shape) - 4.0)
            gate = gate if case["form"] == "log" else gate.exp()
        s["gate"] = gate.to(dtype)
        s["h0"] = randn(states, d) if case["h0"] or case["mode"] == "step" else None
        s["offsets"] = _offsets(gen, n, case["seqs"], dev) if case["seqs"] else None
        leaves = ["u", "gate", "h0"]
        if train:
            s["dy"], s["dlast"] = randn(*shape).to(dtype), randn(states, d)
    s["leaves"] = [k for k in leaves if s[k] is not None]
    if train:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------
_cs2d = None


def _package():
    global _cs2d
    if _cs2d is None:
        path = os.path.join(os.getcwd(), "official-cross-scan_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import cs2d
        _cs2d = cs2d
    return _cs2d


def _run_own(s, case):
    cs2d = _package()
    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "norm":
            x = s["x"].permute(0, 2, 3, 1) if case["layout"] == "image" else s["x"]
            outs = [cs2d.layer_norm(x, s["weight"], s["bias"], s["gate"], _EPS)]
        elif case["mode"] == "step":
            return [cs2d.gated_scan_step(s["u"], s["gate"], s["h0"], form=case["form"], weighted=case["weighted"]), s["h0"]]
        else:
            outs = list(cs2d.gated_scan_1d(s["u"], s["gate"], s["h0"], s["offsets"], form=case["form"], weighted=case["weighted"]))
    if not train:
        return outs
    given = [s["dy"]] + ([s["dlast"]] if case["op"] == "scan" else [])
    return [y.detach() for y in outs] + list(torch.autograd.grad(outs, [s[k] for k in s["leaves"]], given))


# ---- the plain forms -----------------------------------------------------------------------------------------
def _gate_values(gate, form):
    """The factor a, what is left of it to one, and da / dgate."""
    g = gate.float()
    if form == "sigmoid":
        a, c = torch.sigmoid(g), torch.sigmoid(-g)
        return a, c, a * c
    if form == "log":
        a = torch.exp(g)
        return a, -torch.expm1(g), a
    return g, 1.0 - g, torch.ones_like(g)


def _recurrence(a, b):
    """h[t] = a[t] * h[t-1] + b[t] along dim 1, by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], torch.addcmul(b[:, step:], a[:, step:], b[:, :-step])], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _scan_plain(s, case, train):
    dtype = s["u"].dtype
    u, gate = (t.detach().float() for t in (s["u"], s["gate"]))
    a, c, da_dgate = _gate_values(gate, case["form"])
    b = c * u if case["weighted"] else u
    h0 = s["h0"].detach() if s["h0"] is not None else None
    if s["offsets"] is not None:
        total, off = u.shape[0], s["offsets"].long()
        first, last, full = off[:-1].clamp(max=total - 1), (off[1:] - 1).clamp(min=0), (off[1:] > off[:-1]).float()[:, None]
        h0 = torch.zeros(full.shape[0], u.shape[1], device=u.device) if h0 is None else h0
        inside = (torch.arange(total, device=u.device) < off[-1]).float()[:, None]
        cut = torch.zeros(total, 1, device=u.device).index_add_(0, first, full)
        before = torch.zeros_like(u).index_add_(0, first, full * h0)          # the state that a sequence's first row meets
        factor = a * inside * (1.0 - cut)
        h = _recurrence(factor[None], (inside * (b + a * before))[None])[0]
        h_last = torch.where(full > 0, h[last], h0)
        if not train:
            return [h.to(dtype), h_last]
        dlast = s["dlast"]
        g = inside * s["dy"].float() + torch.zeros_like(u).index_add_(0, last, full * dlast)
        ahead = torch.cat([factor[1:], torch.zeros_like(factor[:1])])
        dh = _recurrence(ahead.flip(0)[None], g.flip(0)[None])[0].flip(0)
        prev = before + (1.0 - cut) * torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        dh0 = torch.where(full > 0, a[first] * dh[first], dlast)
    else:
        h0 = torch.zeros(u.shape[0], u.shape[2], device=u.device) if h0 is None else h0
        b = b.clone()
        b[:, 0] += a[:, 0] * h0
        h = _recurrence(a, b)
        if not train:
            return [h.to(dtype), h[:, -1]]
        g = s["dy"].float()
        g[:, -1] += s["dlast"]
        ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        dh = _recurrence(ahead.flip(1), g.flip(1)).flip(1)
        prev = torch.cat([h0[:, None], h[:, :-1]], 1)
        h_last, dh0, inside = h[:, -1], a[:, 0] * dh[:, 0], 1.0
    du = inside * (dh * c if case["weighted"] else dh)
    dgate = inside * dh * (prev - u if case["weighted"] else prev) * da_dgate
    return [h.to(dtype), h_last, du.to(dtype), dgate.to(dtype)] + ([dh0] if s["h0"] is not None else [])


def _step_plain(s, case):
    a, c, _ = _gate_values(s["gate"], case["form"])
    u = s["u"].float()
    s["h0"].copy_(a * s["h0"] + (c * u if case["weighted"] else u))
    return [s["h0"].to(s["u"].dtype), s["h0"]]


def _norm_plain(s, case, train):
    dtype = s["x"].dtype
    x = s["x"].detach().permute(0, 2, 3, 1) if case["layout"] == "image" else s["x"].detach()
    x, weight, bias = x.float(), s["weight"].detach(), s["bias"].detach()
    mid = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((mid * mid).mean(-1, keepdim=True) + _EPS)
    xhat = mid * rstd
    y = xhat * weight + bias
    if s["gate"] is not None:
        z = s["gate"].detach().float()
        sig = torch.sigmoid(z)
        silu = z * sig
        out = y * silu
    else:
        out = y
    if not train:
        return [out.to(dtype)]
    dy = s["dy"].float()
    if s["gate"] is not None:
        dz = dy * y * (sig + silu * (1.0 - sig))
        dy = dy * silu
    dxhat = dy * weight
    dx = rstd * (dxhat - dxhat.mean(-1, keepdim=True) - xhat * (dxhat * xhat).mean(-1, keepdim=True))
    dx = dx.permute(0, 3, 1, 2).contiguous() if case["layout"] == "image" else dx
    dw, db = (dy * xhat).sum((0, 1, 2)), dy.sum((0, 1, 2))
    return [out.to(dtype), dx.to(dtype), dw, db] + ([dz.to(dtype)] if s["gate"] is not None else [])


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    train = case["mode"] == "train"
    with torch.no_grad():
        if case["op"] == "norm":
            return _norm_plain(s, case, train)
        return _step_plain(s, case) if case["mode"] == "step" else _scan_plain(s, case, train)


# ---- the definition in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f = lambda k: s[k].detach().double() if s.get(k) is not None else None
    with torch.no_grad():
        return _norm_exact(case, f) if case["op"] == "norm" else _scan_exact(case, f, s["offsets"])


def _norm_exact(case, f):
    x, weight, bias, gate, dy = f("x"), f("weight"), f("bias"), f("gate"), f("dy")
    if case["layout"] == "image":
        x = x.movedim(1, 3)
    n = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / n
    sd = (((x - mean) ** 2).sum(-1, keepdim=True) / n + _EPS).sqrt()
    norm = (x - mean) / sd
    scaled = norm * weight + bias
    act = gate / (1 + (-gate).exp()) if gate is not None else torch.ones((), dtype=torch.float64, device=x.device)
    out = [scaled * act]
    if dy is None:
        return out
    up = dy * act
    flat = up.reshape(-1, n)
    t = up * weight
    dx = (t - t.sum(-1, keepdim=True) / n - norm * (t * norm).sum(-1, keepdim=True) / n) / sd
    out += [dx.movedim(3, 1) if case["layout"] == "image" else dx, (flat * norm.reshape(-1, n)).sum(0), flat.sum(0)]
    if gate is not None:
        p = 1 / (1 + (-gate).exp())
        out.append(dy * scaled * p * (1 + gate * (1 - p)))
    return out


def _scan_exact(case, f, offsets):
    u, gate, h0, dy, dlast = f("u"), f("gate"), f("h0"), f("dy"), f("dlast")
    if case["form"] == "sigmoid":
        a = 1 / (1 + (-gate).exp())
        slope = a / (1 + gate.exp())
    else:
        a = gate.exp() if case["form"] == "log" else gate
        slope = a if case["form"] == "log" else torch.ones_like(a)
    b = u * (-torch.expm1(gate) if case["form"] == "log" else 1 - a) if case["weighted"] else u
    if case["mode"] == "step":
        h = a * h0 + b
        return [h, h]
    packed = offsets is not None
    rows = u.shape[0] if packed else u.shape[1]
    at = (lambda t, i: t[i]) if packed else (lambda t, i: t[:, i])
    states = case["seqs"] if packed else u.shape[0]
    zero = torch.zeros(states, u.shape[-1], dtype=torch.float64, device=u.device)
    begin = zero if h0 is None else h0
    borders = offsets.tolist() if packed else [0, rows]
    h, prev, last = torch.zeros_like(u), torch.zeros_like(u), begin.clone()
    pieces = [(i, borders[i], borders[i + 1]) for i in range(len(borders) - 1) if borders[i] < borders[i + 1]]
    for i, lo, hi in pieces:
        state = begin[i] if packed else begin
        for t in range(lo, hi):
            at(prev, t).copy_(state)
            state = torch.addcmul(at(b, t), at(a, t), state, out=at(h, t))
        (last[i] if packed else last).copy_(state)
    if dy is None:
        return [h, last]
    du, dgate, dh0 = torch.zeros_like(u), torch.zeros_like(u), dlast.clone()
    dh = torch.zeros_like(u)
    for i, lo, hi in pieces:
        back = dlast[i] if packed else dlast
        for t in range(hi - 1, lo - 1, -1):
            here = torch.add(at(dy, t), back, out=at(dh, t))
            back = here * at(a, t)
        (dh0[i] if packed else dh0).copy_(back)
    if case["weighted"]:
        du = dh * (1 / (1 + gate.exp()) if case["form"] == "sigmoid" else -torch.expm1(gate) if case["form"] == "log" else 1 - a)
        dgate = dh * (prev - u) * slope
    else:
        du, dgate = dh, dh * prev * slope
    return [h, last, du, dgate] + ([dh0] if h0 is not None else [])


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n = case["batch"] * case["h"] * case["w"] * case["dim"]
        tensors = (2 + case["gated"]) + ((2 + case["gated"]) if train else 0)    # x, y (, gate); dy, dx (, dgate)
        return {"bytes": es * n * tensors + 4 * case["dim"] * (4 if train else 2),
                "flops": n * ((8 + 6 * case["gated"]) + ((14 + 12 * case["gated"]) if train else 0))}
    n = case["batch"] * case["length"] * case["dim"]
    state = 4 * case["dim"] * (case["seqs"] or case["batch"])
    states = 1 + bool(case["h0"] or case["mode"] == "step") + ((1 + bool(case["h0"])) if train else 0)
    return {"bytes": es * n * (6 if train else 3) + state * states, "flops": n * (6 + 2 * case["weighted"] + (12 if train else 0))}
