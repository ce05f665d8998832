"""Workloads of the layer norm, top-logit distillation and microscaled 4-bit operators.

Each case is one pass as a training loop or an acting loop makes it.  ``run`` computes it from elementary tensor operations
(``own`` false) or through this package's operators (``own`` true); ``exact`` gives the same results from the definitions in
64 bits.  Element types are named "f32", "bf16" and "f16".
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-5


def listed():
    return [
        # one acting step of 16 environments through one block of the default width: latency
        dict(name="norm_step", op="norm", rows=16, width=512, dtype="f32", wdtype="f32", train=False, stride=512),
        # one block of the default update, 16 sequences of 64 steps, forward and backward
        dict(name="norm_update", op="norm", rows=1024, width=512, dtype="f32", wdtype="f32", train=True, stride=512),
        # a wide block over a large batch in bfloat16, weights held in fp32
        dict(name="norm_wide", op="norm", rows=16384, width=4096, dtype="bf16", wdtype="f32", train=True, stride=4096),
        # the critic's 255 buckets at the 16 x 15 imagined states, the teacher's 16 largest of them
        dict(name="distill_buckets", op="distill", rows=240, vocab=255, k=16, dtype="f32", temperature=1.0, rest=False, ragged=False,
             masked=False),
        # a large vocabulary over a training batch, teacher stored with its log-sum-exp, softened
        dict(name="distill_batch", op="distill", rows=4096, vocab=32768, k=64, dtype="bf16", temperature=2.0, rest=True,
             ragged=True, masked=False),
        # a handful of rows over a very long, odd vocabulary with forbidden entries
        dict(name="distill_long", op="distill", rows=5, vocab=128001, k=100, dtype="f16", temperature=1.0, rest=False, ragged=True,
             masked=True),
        # activations of the wide model's update to 4 bits and back
        dict(name="quantise_rows", op="quantise", rows=1024, width=4096, dtype="f32"),
        # a wide model's recurrent weight to 4 bits and back, in bfloat16
        dict(name="quantise_weight", op="quantise", rows=12288, width=4096, dtype="bf16"),
        # the wide model's recurrent product at one step of 16 trajectories: the weight is streamed once
        dict(name="linear_step", op="linear", rows=16, out=12288, width=4096, dtype="bf16", bias=True, train=False),
        # 16 x 64 rows through a frozen 4-bit layer of the wide model, with the gradient that flows back through it
        dict(name="linear_update", op="linear", rows=1024, out=4096, width=4096, dtype="bf16", bias=True, train=True),
        # both operands in 4 bits: a ragged small product and a large one
        dict(name="product_ragged", op="product", rows=257, out=1000, width=4080, dtype="f32", bias=True),
        dict(name="product_large", op="product", rows=8192, out=8192, width=8192, dtype="bf16", bias=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "distill", "distill", "quantise", "linear", "linear", "product"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        width = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, max(1, min(16384, 2 ** 26 // width)))
        return dict(op=op, rows=rows, width=width, dtype=dtype, wdtype=rng.choice(["f32", dtype]), train=rng.random() < 0.6,
                    stride=width + rng.choice([0, 0, 1, 8, 40]))
    if op == "distill":
        vocab = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, 2 ** 26 // vocab)))
        k = _log_int(rng, 1, min(vocab, 128))
        return dict(op=op, rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=rng.choice([0.5, 1.0, 2.0, 4.0]),
                    rest=rng.random() < 0.5, ragged=rng.random() < 0.5, masked=rng.random() < 0.3)
    if op == "quantise":
        return dict(op=op, rows=_log_int(rng, 1, 12288), width=_log_int(rng, 1, 4096), dtype=dtype)
    if op == "linear":
        return dict(op=op, rows=_log_int(rng, 1, 2048), out=_log_int(rng, 8, 8192), width=_log_int(rng, 8, 4096), dtype=dtype,
                    bias=rng.random() < 0.5, train=rng.random() < 0.5)
    return dict(op=op, rows=_log_int(rng, 1, 8192), out=_log_int(rng, 8, 8192), width=_log_int(rng, 8, 8192), dtype=dtype,
                bias=rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _rows_like_activations(rows, width, g):
    """Unit-scale rows with a few loud columns and an offset per row, as pre-activations have."""
    x = torch.randn(rows, width, generator=g, device=DEV)
    loud = torch.randint(0, width, (max(1, width // 128),), generator=g, device=DEV)
    x[:, loud] *= 8.0
    return x + 0.5 * torch.randn(rows, 1, generator=g, device=DEV)


def _weight4(out, width, g):
    """A weight as it is stored in 4 bits: codes (out, blocks * 16), scale bytes (out, blocks)."""
    w = torch.randn(out, width, generator=g, device=DEV) / math.sqrt(width)
    return _pack(*_codes(w))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 17)
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    st = dict(case=case)
    if op == "norm":
        rows, width = case["rows"], case["width"]
        full = _rows_like_activations(rows, case["stride"], g).to(dt)
        st["x"] = full[:, :width].requires_grad_(case["train"])
        st["w"] = (1.0 + 0.2 * torch.randn(width, generator=g, device=DEV)).to(DTYPES[case["wdtype"]]).requires_grad_(case["train"])
        st["b"] = (0.2 * torch.randn(width, generator=g, device=DEV)).to(DTYPES[case["wdtype"]]).requires_grad_(case["train"])
        if case["train"]:
            st["dy"] = torch.randn(rows, width, generator=g, device=DEV).to(dt)
    elif op == "distill":
        rows, vocab, k, t = case["rows"], case["vocab"], case["k"], case["temperature"]
        teacher = 2.5 * torch.randn(rows, vocab, generator=g, device=DEV)
        logits = (0.6 * teacher + 1.5 * torch.randn(rows, vocab, generator=g, device=DEV)).to(dt)
        values, indices = teacher.topk(k, dim=1)
        lse = torch.logsumexp(teacher.double() / t, dim=1).float()
        if case["masked"]:   # entries the student may not choose; the teacher's own stay open
            off = torch.rand(rows, vocab, generator=g, device=DEV) < 0.25
            off.scatter_(1, indices, False)
            logits = logits.masked_fill(off, float("-inf"))
        if case["ragged"]:   # lists of different lengths, some of them empty
            have = torch.randint(0, k + 1, (rows, 1), generator=g, device=DEV)
            indices = indices.masked_fill(torch.arange(k, device=DEV) >= have, -1)
        st.update(logits=logits.requires_grad_(True), values=values, indices=indices, lse=lse if case["rest"] else None,
                  g=torch.rand(rows, generator=g, device=DEV) * (1024.0 if dt is torch.float16 else 1.0))   # fp16: a scaled loss
    elif op == "quantise":
        st["x"] = _rows_like_activations(case["rows"], case["width"], g).to(dt)
    else:
        rows, out, width = case["rows"], case["out"], case["width"]
        train = case.get("train", False)
        st["x"] = _rows_like_activations(rows, width, g).to(dt).requires_grad_(train)
        codes, scales = _weight4(out, width, g)
        st["codes"], st["scales"] = codes, scales
        if own:
            from dreamer_amd import mx4
            st["w4"] = mx4.MX4Tensor(codes, scales, width)
        st["b"] = (0.1 * torch.randn(out, generator=g, device=DEV)).to(dt).requires_grad_(train) if case["bias"] else None
        if train:
            st["dy"] = torch.randn(rows, out, generator=g, device=DEV).to(dt)
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _codes(x):
    """4-bit codes (rows, blocks, 32) and scale bytes (rows, blocks) of a float matrix, blocks of 32 along a row."""
    rows, width = x.shape
    nb = (width + 31) // 32
    v = x.float()
    if nb * 32 != width:
        v = torch.cat([v, torch.zeros(rows, nb * 32 - width, device=x.device)], dim=1)
    v = v.view(rows, nb, 32)
    top = v.abs().amax(dim=2)
    e = torch.where(top > 0, torch.frexp(top)[1] - 1 - 2, torch.full_like(top, -127, dtype=torch.int32)).clamp(-127, 127)
    a = torch.ldexp(v.abs(), -e.unsqueeze(2))
    # nearest, ties to the even code: up to the middle inclusive where the upper code is odd
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
            + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8))
    return code | (torch.signbit(v).to(torch.uint8) << 3), (e + 127).to(torch.uint8)


def _pack(codes, scales):
    rows, nb, _ = codes.shape
    return (codes[:, :, 0::2] | (codes[:, :, 1::2] << 4)).reshape(rows, nb * 16), scales


def _values(codes, scales, width):
    """fp32 values of unpacked codes and their scale bytes."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = torch.ldexp(table[codes.long()], (scales.int() - 127).unsqueeze(2))
    return v.reshape(codes.shape[0], -1)[:, :width]


def _unpack(packed):
    rows = packed.shape[0]
    return torch.stack([packed & 15, packed >> 4], dim=2).view(rows, -1, 32)


def _norm_plain(st):
    case = st["case"]
    x, w, b = st["x"].detach().float(), st["w"].detach().float(), st["b"].detach().float()
    mean = x.mean(dim=1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(dim=1, keepdim=True) + EPS)
    xh = xc * rstd
    dt, wt = st["x"].dtype, st["w"].dtype
    y = (xh * w + b).to(dt)
    if not case["train"]:
        return {"y": y}
    dy = st["dy"].float()
    gy = dy * w
    dx = rstd * (gy - gy.mean(dim=1, keepdim=True) - xh * (gy * xh).mean(dim=1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dw": (dy * xh).sum(dim=0).to(wt), "db": dy.sum(dim=0).to(wt)}


def _distill_plain(st):
    # the teacher's probabilities, the row sums and scalars in 64 bits: 1 - sum p, log Q and the gradient's factors are differences
    t = st["case"]["temperature"]
    s = st["logits"].detach().float()
    idx = st["indices"]
    rows, vocab = s.shape
    here = (idx >= 0) & (idx < vocab)
    safe = torch.where(here, idx, torch.zeros_like(idx))
    none = ~here.any(dim=1)
    top = torch.where(here, st["values"].double() / t, torch.full_like(st["values"], float("-inf"), dtype=torch.float64))
    m = s.amax(dim=1, keepdim=True)
    ex = torch.exp((s - m) / t)
    z = ex.sum(dim=1, dtype=torch.float64)
    logq = (torch.gather(s, 1, safe).double() - m.double()) / t - torch.log(z).unsqueeze(1)
    if st["lse"] is None:
        tm = torch.where(none, torch.zeros_like(top[:, 0]), top.amax(dim=1)).unsqueeze(1)
        p = torch.exp(top - tm)
        p = p / torch.where(none.unsqueeze(1), torch.ones_like(tm), p.sum(dim=1, keepdim=True))
    else:
        p = torch.exp(top - st["lse"].double().unsqueeze(1))
    loss = torch.where(p > 0, p * (torch.log(p) - logq), torch.zeros_like(p)).sum(dim=1)
    total = p.sum(dim=1)
    factor = torch.where(none, torch.zeros_like(total), st["g"].double() / t)
    listed_p = torch.zeros_like(s).scatter_add_(1, safe, (p * factor.unsqueeze(1)).float())
    if st["lse"] is None:
        ds = ex * (factor * total / z).float().unsqueeze(1) - listed_p
    else:
        out = torch.zeros(rows, vocab, dtype=torch.int32, device=s.device).scatter_add_(1, safe, here.int()) == 0
        zr = torch.where(out, ex, torch.zeros_like(ex)).sum(dim=1, dtype=torch.float64)
        rest = torch.where(zr > 0, (1.0 - total).clamp_min(0.0), torch.zeros_like(total))
        live = rest > 0
        loss = loss + torch.where(live, rest * (torch.log(rest) - torch.log(zr / z)), torch.zeros_like(rest))
        inside = factor * (total + rest) / z
        outside = inside - torch.where(live, factor * rest / zr, torch.zeros_like(rest))
        ds = ex * torch.where(out, outside.float().unsqueeze(1), inside.float().unsqueeze(1)) - listed_p
    return {"loss": torch.where(none, torch.zeros_like(loss), loss).float(), "dlogits": ds.to(st["logits"].dtype)}


def _linear_plain(st):
    case = st["case"]
    dt = st["x"].dtype
    w = _values(_unpack(st["codes"]), st["scales"], case["width"])
    x = st["x"].detach().float()
    if case["op"] == "product":
        x = _values(*_codes(x), case["width"])
    y = x @ w.t()
    if st["b"] is not None:
        y = y + st["b"].detach().float()
    out = {"y": y.to(dt)}
    if case.get("train", False):
        dy = st["dy"].float()
        out["dx"] = (dy @ w).to(dt)
        if st["b"] is not None:
            out["db"] = dy.sum(dim=0).to(dt)
    return out


def _plain(st):
    op = st["case"]["op"]
    if op == "norm":
        return _norm_plain(st)
    if op == "distill":
        return _distill_plain(st)
    if op == "quantise":
        return {"values": _values(*_codes(st["x"]), st["case"]["width"]).to(st["x"].dtype)}
    return _linear_plain(st)


# ---- the package's operators --------------------------------------------------------------------------------------------

def _own(st):
    from dreamer_amd import losses, mx4, norm
    case = st["case"]
    op = case["op"]
    if op == "norm":
        y = norm.layer_norm(st["x"], st["w"], st["b"], EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "distill":
        loss = losses.distill_topk_rows(st["logits"], st["values"], st["indices"], case["temperature"], st["lse"])
        return {"loss": loss, "dlogits": torch.autograd.grad(loss, st["logits"], st["g"])[0]}
    if op == "quantise":
        return {"values": mx4.quantize(st["x"]).dequantize(st["x"].dtype)}
    if op == "product":
        return {"y": mx4.linear(mx4.quantize(st["x"]), st["w4"], st["b"], out_dtype=st["x"].dtype)}
    y = mx4.linear(st["x"], st["w4"], st["b"])
    out = {"y": y}
    if case["train"]:
        if st["b"] is None:
            out["dx"] = torch.autograd.grad(y, st["x"], st["dy"])[0]
        else:
            out["dx"], out["db"] = torch.autograd.grad(y, (st["x"], st["b"]), st["dy"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_values(x):
    """Values that a float matrix takes in 4 bits: each element goes to the nearest of the 15 numbers, found by distance; of
    two as near the one with the even place in the table."""
    rows, width = x.shape
    res = torch.empty(rows, width, dtype=torch.float64, device=x.device)
    table = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    for c in range(0, width, 32):
        v = x[:, c:c + 32].double()
        top = v.abs().max(dim=1, keepdim=True).values
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -200)))
        e = e - (torch.pow(2.0, e) > top).double() + (torch.pow(2.0, e + 1) <= top).double()
        unit = torch.pow(2.0, (e - 2).clamp(-127, 127))
        near = (v.abs() / unit).clamp_max(6.0).unsqueeze(-1).sub(table).abs()
        best = near.min(dim=-1, keepdim=True).values
        even = (near == best) & (torch.arange(8, device=x.device) % 2 == 0)
        pick = torch.where(even.any(dim=-1), even.double().argmax(dim=-1), near.argmin(dim=-1))
        res[:, c:c + 32] = torch.sign(v) * table[pick] * unit
    return res


def _exact_weight(packed, scales, width):
    n = packed.long()
    nib = torch.empty(n.shape[0], 2 * n.shape[1], dtype=torch.long, device=n.device)
    nib[:, 0::2] = n % 16
    nib[:, 1::2] = n // 16
    mag = torch.tensor(E2M1, dtype=torch.float64, device=n.device)[nib % 8]
    unit = torch.pow(2.0, scales.double() - 127.0).repeat_interleave(32, dim=1)
    return (torch.where(nib >= 8, -mag, mag) * unit)[:, :width]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, w, b = st["x"].detach().double(), st["w"].detach().double(), st["b"].detach().double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        xh = (x - mean) / sd
        res = {"y": w * xh + b}
        if case["train"]:
            dy = st["dy"].double()
            wd = w * dy
            n = case["width"]
            res["dx"] = (n * wd - wd.sum(1, keepdim=True) - xh * (wd * xh).sum(1, keepdim=True)) / (n * sd)
            res["dw"] = (xh * dy).sum(0)
            res["db"] = dy.sum(0)
        return res
    if op == "distill":
        rows, vocab = case["rows"], case["vocab"]
        t = case["temperature"]
        loss = torch.zeros(rows, dtype=torch.float64, device=DEV)
        grad = torch.zeros(rows, vocab, dtype=torch.float64, device=DEV)
        idx, val = st["indices"], st["values"].double()
        step = max(1, 2 ** 24 // vocab)
        for r0 in range(0, rows, step):
            sl = slice(r0, min(rows, r0 + step))
            logq = torch.log_softmax(st["logits"].detach()[sl].double() / t, dim=1)
            n = logq.shape[0]
            ok = idx[sl] >= 0
            tv = (val[sl] / t).masked_fill(~ok, float("-inf"))
            base = torch.logsumexp(tv, dim=1) if st["lse"] is None else st["lse"][sl].double()
            p = torch.zeros(n, vocab + 1, dtype=torch.float64, device=DEV)   # the last column takes absent entries
            p.scatter_(1, torch.where(ok, idx[sl], vocab), torch.where(ok, torch.exp(tv - base.unsqueeze(1)), 0.0))
            seen = torch.zeros(n, vocab + 1, dtype=torch.bool, device=DEV)
            seen.scatter_(1, torch.where(ok, idx[sl], vocab), True)
            p, seen = p[:, :vocab], seen[:, :vocab]
            cost = torch.special.xlogy(p, p).sum(1) - torch.where(p > 0, p * logq, 0.0).sum(1)
            total = p.sum(1)
            d = -p
            if st["lse"] is not None:
                inside = logq.masked_fill(seen, float("-inf"))
                log_rest = torch.logsumexp(inside, dim=1)
                left = torch.where(torch.isfinite(log_rest), (1.0 - total).clamp_min(0.0), 0.0)
                on = left > 0
                cost = cost + torch.where(on, torch.special.xlogy(left, left) - left * log_rest, 0.0)
                d = d - torch.where(on.unsqueeze(1), left.unsqueeze(1) * torch.exp(inside - log_rest.unsqueeze(1)), 0.0)
                total = total + left
            d = d + total.unsqueeze(1) * torch.exp(logq)
            some = ok.any(dim=1)
            loss[sl] = torch.where(some, cost, 0.0)
            grad[sl] = torch.where(some.unsqueeze(1), d * (st["g"][sl].double() / t).unsqueeze(1), 0.0)
        return {"loss": loss, "dlogits": grad}
    if op == "quantise":
        return {"values": _exact_values(st["x"])}
    w = _exact_weight(st["codes"], st["scales"], case["width"])
    x = st["x"].detach()
    x = _exact_values(x) if op == "product" else x.double()
    y = torch.matmul(x, w.transpose(0, 1).contiguous())
    res = {"y": y if st["b"] is None else y + st["b"].detach().double()}
    if case.get("train", False):
        res["dx"] = torch.matmul(st["dy"].double(), w)
        if st["b"] is not None:
            res["db"] = st["dy"].double().sum(0)
    return res


def work(case):
    """Bytes each input read once and each output written once, and the operations of the products and row sums."""
    s = SIZE[case["dtype"]]
    rows = case["rows"]
    op = case["op"]
    if op == "norm":
        n = rows * case["width"]
        ws = SIZE[case["wdtype"]] * case["width"]
        if not case["train"]:
            return {"bytes": 2 * n * s + 2 * ws, "flops": 8 * n}
        return {"bytes": 5 * n * s + 4 * ws, "flops": 25 * n}      # x read by both directions, y written, dy read, dx written
    if op == "distill":
        n = rows * case["vocab"]
        lists = rows * case["k"] * 12 + rows * (12 if case["rest"] else 8)
        return {"bytes": 3 * n * s + lists, "flops": 12 * n}       # logits read by both directions, their gradient written
    nb = (case["width"] + 31) // 32
    if op == "quantise":
        n = rows * case["width"]
        return {"bytes": 2 * n * s + rows * nb * 17, "flops": 4 * n}
    out, width = case["out"], case["width"]
    passes = 2 if case.get("train", False) else 1
    wbytes = out * nb * 17
    return {"bytes": passes * (rows * width * s + rows * out * s + wbytes) + (s * out if case["bias"] else 0),
            "flops": passes * 2 * rows * out * width}
