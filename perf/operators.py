"""Cases of the 8-bit operators: the matrix product in 8-bit integers with a
scale per token and per channel, alone and as the backbone of the multi-LoRA
linear, and activations kept in 8 bits for the backward pass.

    q(x)[i, k]  = round(x[i, k] / s[i]),  s[i] = float32(max_k |x[i, k]| / 127)
    linear      y  = s_x[i] s_w[j] sum_k q(x)[i, k] q(w)[j, k] + bias[j]
                dx = s_g[i] sum_j q(g)[i, j] q(w)[j, k],  g[i, j] = float32(dy[i, j] s_w[j])
    lora        y += c (x A^T) B^T on the rows of each adapter, with
                dz = c dy B, dx += dz A, dB = c dy^T (x A^T) and
                dA = dz^T x, or with saved 8-bit rows dA = dz^T (s_x q(x))
    save        x kept as q(x), s and read back as s_x q(x)

Ties of the rounding go to the even integer and a row of zeros has s = 0.
Where ``own`` is false the operators are computed in plain torch operations;
where it is true through the package's calls.
"""

import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-tlora-reproduction_b200")
    if src not in sys.path:
        sys.path.insert(0, src)
    import tlora_b200

    return tlora_b200


def _linear(name, rows, d_in, d_out, dtype, bias=True, grad=False):
    return {"name": name, "op": "linear", "rows": rows, "d_in": d_in, "d_out": d_out, "dtype": dtype, "bias": bias,
            "grad": grad}


def _lora(name, rows, d_in, d_out, dtype, adapters, ranks, split, mixed=False, unknown=False, base8=True,
          save8=True, grad=True):
    return {"name": name, "op": "lora", "rows": rows, "d_in": d_in, "d_out": d_out, "dtype": dtype,
            "adapters": adapters, "ranks": ranks, "split": split, "mixed": mixed, "unknown": unknown,
            "base8": base8, "save8": save8, "grad": grad}


def _save(name, rows, d_in, dtype):
    return {"name": name, "op": "save", "rows": rows, "d_in": d_in, "dtype": dtype}


def listed():
    return [
        # one token of a served request through a square projection: latency alone
        _linear("linear_one_token", 1, 4096, 4096, "bf16"),
        # a small batch of tokens through an MLP up-projection: the weights are the bytes
        _linear("linear_eight_tokens", 8, 4096, 11008, "bf16", bias=False),
        # a ragged batch through a layer of odd sizes, in 32 bits
        _linear("linear_ragged", 777, 1000, 1531, "fp32"),
        # a long prompt, or a layer without adapters in training: product and input gradient
        _linear("linear_prompt_grad", 8192, 4096, 11008, "fp16", grad=True),
        # sixteen requests of sixteen adapters, one token each, in arrival order, one of them without an adapter
        _lora("lora_sixteen_tokens", 16, 4096, 4096, "bf16", 16, "8,16,32,64", 5, mixed=True, unknown=True,
              save8=False, grad=False),
        # prompts of sixteen jobs packed into one batch, answered (no gradients)
        _lora("lora_packed_forward", 18432, 4096, 4096, "bf16", 16, "8,16,32,64", 1, save8=False, grad=False),
        # a training step of an MLP up-projection shared by eight jobs
        _lora("lora_up_projection_step", 65536, 4096, 11008, "bf16", 8, "16,64", 2),
        # a training step with small ragged jobs, odd ranks and rows of no job, rows in arrival order
        _lora("lora_ragged_step", 3001, 1048, 776, "fp16", 7, "1,5,33,64,65,130", 3, mixed=True, unknown=True),
        # the small 32-bit configuration: four jobs in a square layer
        _lora("lora_small_fp32_step", 640, 1024, 1024, "fp32", 4, "4,8,16,32", 4),
        # a 16-bit backbone whose inputs are kept in 8 bits until the backward pass
        _lora("lora_saved_inputs_step", 18432, 4096, 4096, "bf16", 16, "8,16,32,64", 6, base8=False),
        # keeping the activations of a short ragged batch, and reading them back
        _save("save_ragged", 257, 1000, "fp16"),
        # the same for the batch of the up-projection's training step
        _save("save_long", 65536, 4096, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["linear", "linear", "lora", "lora", "save"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = _log(rng, 1, 8192 if dtype == "fp32" else 65536)
    if op == "save":
        return {k: v for k, v in _save("", rows, _log(rng, 64, 8192 if rows < 32768 else 4096), dtype).items()
                if k != "name"}
    d_in, d_out = _log(rng, 64, 4096), _log(rng, 64, 11008)
    if rng.random() < 0.5:
        d_in, d_out = (d_in + 63) // 64 * 64, (d_out + 63) // 64 * 64
    if op == "linear":
        c = _linear("", min(rows, 16384), d_in, d_out, dtype, rng.random() < 0.5, rng.random() < 0.5)
    else:
        # layers with adapters have features in multiples of 8
        d_in, d_out = (d_in + 7) // 8 * 8, (d_out + 7) // 8 * 8
        if dtype == "fp32":
            d_in, d_out, rows = min(d_in, 1024), min(d_out, 1024), min(rows, 2048)
        n = rng.randint(1, 16)
        ranks = ",".join(str(rng.choice([1, 4, 8, 16, 24, 32, 64, 100])) for _ in range(4))
        base8 = rng.random() < 0.7
        grad = rng.random() < 0.7
        c = _lora("", rows, d_in, d_out, dtype, n, ranks, rng.randint(0, 10 ** 6), rng.random() < 0.4,
                  rng.random() < 0.3, base8, grad and (not base8 or rng.random() < 0.6), grad)
        if not base8 and not grad:
            c["base8"] = True
    del c["name"]
    return c


def _jobs(case):
    """Ranks and row counts of the adapters, and the rows that name none."""
    r = random.Random(case["split"])
    choices = [int(v) for v in case["ranks"].split(",")]
    n, rows = case["adapters"], case["rows"]
    ranks = [choices[i % len(choices)] for i in range(n)]
    none = max(1, rows // 16) if case["unknown"] and rows > 1 else 0
    left = rows - none
    if left <= n:
        counts = [1 if i < left else 0 for i in range(n)]
    else:
        w = [0.25 + r.random() for _ in range(n)]
        counts = [int(left * v / sum(w)) for v in w]
        counts[r.randrange(n)] += left - sum(counts)
    return ranks, counts, none


def _draws(shape, g, dev, scale=1.0):
    return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(scale)


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    rows, d_in = case["rows"], case["d_in"]
    # activations: N(0, 1) with a few channels several times larger, tokens of different size
    chan = torch.where(torch.rand(d_in, generator=g, device=dev) < 0.01, 6.0, 1.0)
    tok = torch.exp(0.4 * torch.randn(rows, 1, generator=g, device=dev))
    s = {"case": case, "x": _draws((rows, d_in), g, dev).mul_(chan).mul_(tok).to(dt)}
    if case["op"] == "save":
        return s
    d_out = case["d_out"]
    s["w"] = _draws((d_out, d_in), g, dev, d_in ** -0.5).to(dt)
    s["bias"] = _draws((d_out,), g, dev, 0.1).to(dt) if case.get("bias", True) else None
    if case["grad"]:
        tok = torch.exp(0.7 * torch.randn(rows, 1, generator=g, device=dev))
        s["dy"] = _draws((rows, d_out), g, dev, 0.01).mul_(tok).to(dt)
    if case["op"] == "linear":
        return s
    ranks, counts, none = _jobs(case)
    ids = torch.cat([torch.full((c,), i, dtype=torch.int64) for i, c in enumerate(counts)] +
                    [torch.full((none,), -1, dtype=torch.int64)])
    if case["mixed"]:
        ids = ids[torch.randperm(rows, generator=torch.Generator().manual_seed(seed))]
    s["ids"] = ids
    s["A"] = [((torch.rand(r, d_in, generator=g, device=dev) * 2 - 1) * d_in ** -0.5).to(dt) for r in ranks]
    s["B"] = [_draws((d_out, r), g, dev, 0.02).to(dt) for r in ranks]
    s["active"] = [i for i, c in enumerate(counts) if c > 0]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "save":
        return s
    x, w = s["x"], s["w"]
    if own and case["grad"]:
        x.requires_grad_(True)
    if case["op"] == "linear":
        if own:
            s["weight"] = _package().ops.quantize_rows(w)
        else:
            s["wq"], s["ws"] = _quantize(w)
        return s
    if not own:
        s["rows_of"] = [(s["ids"] == i).nonzero().squeeze(1).to(x.device) for i in range(case["adapters"])]
        if case["base8"]:
            s["wq"], s["ws"] = _quantize(w)
        return s
    ranks = _jobs(case)[0]
    with torch.device(x.device):
        m = _package().MultiLoRALinear(case["d_in"], case["d_out"], {i: r for i, r in enumerate(ranks)}).to(x.dtype)
    with torch.no_grad():
        m.base.weight.copy_(w)
        m.base.bias.copy_(s["bias"])
        for i in range(len(ranks)):
            ad = m.adapters[str(i)]
            ad.alpha, ad.scaling = 2.0 * ranks[i], 2.0
            ad.A.copy_(s["A"][i])
            ad.B.copy_(s["B"][i])
    if case["base8"]:
        m.quantize_base()
    if case["save8"]:
        m.save_input = "int8"
    # the routing of a batch is the same for every layer and pass: planned once
    s["model"], s["plan"] = m, m.route(s["ids"])
    m.make_resident(s["plan"])
    if case["grad"]:
        s["wanted"] = [x] + [p for i in s["active"] for p in (m.adapters[str(i)].A, m.adapters[str(i)].B)]
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case = s["case"]
    ops = _package().ops
    if case["op"] == "save":
        kept = ops.quantize_rows(s["x"])
        return {"x": ops.dequantize_rows(kept, s["x"].dtype), "scale": kept.scale}
    if not case["grad"]:
        with torch.no_grad():
            if case["op"] == "linear":
                return {"y": ops.int8_linear(s["x"], s["weight"], s["bias"])}
            return {"y": s["model"](s["x"], s["ids"], plan=s["plan"])}
    if case["op"] == "linear":
        y = ops.int8_linear(s["x"], s["weight"], s["bias"])
        dx, = torch.autograd.grad(y, [s["x"]], s["dy"])
        return {"y": y.detach(), "dx": dx}
    y = s["model"](s["x"], s["ids"], plan=s["plan"])
    g = torch.autograd.grad(y, s["wanted"], s["dy"])
    return {"y": y.detach(), "dx": g[0], "da": list(g[1::2]), "db": list(g[2::2])}


# ---- the plain form: products, sums and comparisons in 32 bits

def _quantize(x):
    """8-bit rows as (integers in float32, scales): the quotients next to a
    rounding border are decided in 64 bits."""
    s = x.float().abs().amax(1)
    s = s / torch.full_like(s, 127.0)  # a quotient (by a plain number it would be a product with the reciprocal)
    d = torch.where(s > 0, s, torch.ones_like(s)).double()[:, None]
    q = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    step = max(1, (1 << 27) // x.shape[1])
    for i in range(0, x.shape[0], step):
        q[i:i + step] = torch.round(x[i:i + step].double() / d[i:i + step])
    return q, s


def _run_plain(s):
    case, x = s["case"], s["x"]
    dt = x.dtype
    if case["op"] == "save":
        q, sx = _quantize(x)
        return {"x": (q * sx[:, None]).to(dt), "scale": sx}
    base8 = case["op"] == "linear" or case["base8"]
    xf = x.float()
    if base8 or case.get("save8"):
        xq, sx = _quantize(x)
    if base8:
        y = (xq @ s["wq"].t()).mul_(sx[:, None]).mul_(s["ws"])
    else:
        y = xf @ s["w"].float().t()
    if s["bias"] is not None:
        y += s["bias"].float()
    if case["op"] == "lora":
        u = {}
        for i in s["active"]:
            r = s["rows_of"][i]
            u[i] = xf[r] @ s["A"][i].float().t()
            y[r] += 2.0 * (u[i] @ s["B"][i].float().t())
    out = {"y": y.to(dt)}
    if not case["grad"]:
        return out
    dy = s["dy"].float()
    if base8:
        gq, sg = _quantize(dy * s["ws"])
        dx = (gq @ s["wq"]).mul_(sg[:, None])
        del gq
    else:
        dx = dy @ s["w"].float()
    if case["op"] == "lora":
        da, db = [], []
        if case["save8"]:
            xf = xq.mul_(sx[:, None])
        for i in s["active"]:
            r = s["rows_of"][i]
            dz = 2.0 * (dy[r] @ s["B"][i].float())
            dx[r] += dz @ s["A"][i].float()
            da.append((dz.t() @ xf[r]).to(dt))
            db.append((2.0 * (dy[r].t() @ u[i])).to(dt))
        out["da"], out["db"] = da, db
    out["dx"] = dx.to(dt)
    return out


# ---- the definition in 64 bits

def _rows8(v):
    """float64 values -> the float64 values that their 8-bit rows stand for.
    The scale is part of the stored form and is a float32 number."""
    top = v.abs().max(dim=1, keepdim=True).values
    unit = (top / torch.full_like(top, 127.0)).to(torch.float32).to(torch.float64)
    safe = unit.masked_fill(unit == 0, 1.0)
    return v.div(safe).round_().mul_(unit), unit.squeeze(1)


def exact(case, seed):
    state = _inputs(case, seed)
    x = state["x"].double()
    if case["op"] == "save":
        v, unit = _rows8(x)
        return {"x": v, "scale": unit}
    eight = case["op"] == "linear" or case["base8"]
    kept = _rows8(x)[0] if eight or case.get("save8") else x
    w = state["w"].double()
    if eight:
        w, unit_w = _rows8(w)
    y = torch.matmul(kept if eight else x, w.transpose(0, 1))
    if state["bias"] is not None:
        y = y + state["bias"].double()
    out = {"y": y}
    dy = state["dy"].double() if case["grad"] else None
    if dy is not None:
        if eight:
            # the scaled gradient is formed in float32 before its 8-bit rows are
            g = (state["dy"].float() * unit_w.float()).double()
            w = w.div(unit_w.masked_fill(unit_w == 0, 1.0)[:, None]).round_()
            out["dx"] = torch.matmul(_rows8(g)[0], w)
            del g
        else:
            out["dx"] = torch.matmul(dy, w)
    if case["op"] == "linear":
        return out
    ids = state["ids"].to(x.device)
    das, dbs = [], []
    for i in state["active"]:
        mine = ids == i
        a, b = state["A"][i].double(), state["B"][i].double()
        low = torch.matmul(x[mine], a.transpose(0, 1))
        y[mine] += 2.0 * torch.matmul(low, b.transpose(0, 1))
        if dy is not None:
            back = 2.0 * torch.matmul(dy[mine], b)
            out["dx"][mine] += torch.matmul(back, a)
            das.append(torch.matmul(back.transpose(0, 1), (kept if case["save8"] else x)[mine]))
            dbs.append(2.0 * torch.matmul(dy[mine].transpose(0, 1), low))
    if dy is not None:
        out["da"], out["db"] = das, dbs
    return out


def work(case):
    rows, d_in = case["rows"], case["d_in"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "save":
        # read once, kept in 8 bits with a scale per row, read back
        return {"bytes": rows * (2 * d_in * e + 2 * d_in + 8), "flops": 3 * rows * d_in}
    d_out = case["d_out"]
    base8 = case["op"] == "linear" or case["base8"]
    w = d_in * d_out * (1 if base8 else e) + (4 * d_out if base8 else 0)
    passes = 2 if case["grad"] else 1
    nbytes = passes * (w + rows * (d_in + d_out) * e) + d_out * e
    flops = passes * 2 * rows * d_in * d_out
    if case["op"] == "lora":
        ranks, counts, _ = _jobs(case)
        used = sum(r for r, c in zip(ranks, counts) if c)
        rsum = sum(r * c for r, c in zip(ranks, counts))
        nbytes += (2 if case["grad"] else 1) * used * (d_in + d_out) * e
        flops += 2 * rsum * (d_in + d_out) * (3 if case["grad"] else 1)
        if case["save8"]:
            nbytes += 2 * rows * (d_in + 4)
    return {"bytes": nbytes, "flops": flops}
