"""What is measured of the coordinator-side operators that take a block's output to the next block and to the
answer: the block join (rank sum, norm after the block, gate, residual, norm before the next block, wire rows),
products with MXFP4 weights for few rows, and token log probabilities with entropy and top alternatives.

`run` computes them in elementary torch operations, or, where `own` is set, through the package's entry points.
"""
import math

import torch

own = False

WIRE_BLOCK = 32  # values per shared scale, in wire rows and in the weights alike
EPS = 1e-5


def listed():
    return [
        # one decoded token between two blocks: launch latency
        dict(name="join_token", op="join", rows=1, cols=4096, planes=1, post=False, gate="none", wire=False),
        # a decode batch whose routed sum arrives as the four ranks' rows; its wire rows go into the next request frame
        dict(name="join_decode_ranks", op="join", rows=128, cols=4096, planes=4, post=False, gate="none", wire=True),
        # rows that no vector load divides, norms on both sides of the block, a gate value for each token
        dict(name="join_odd", op="join", rows=1021, cols=2047, planes=2, post=True, gate="row", wire=False),
        # a prefill chunk: norms on both sides, a gate for each channel, both forms of the normed row
        dict(name="join_prefill", op="join", rows=8192, cols=4096, planes=1, post=True, gate="column", wire=True),
        # a projection of the hidden size for one token: latency again
        dict(name="w4_token", op="w4", rows=1, n=4096, k=4096, x="bf16", y="bf16"),
        # router logits of a small batch: few weight rows, so the work has to be spread along k
        dict(name="w4_router", op="w4", rows=16, n=256, k=4096, x="bf16", y="f32"),
        # odd sizes, on wire rows
        dict(name="w4_odd", op="w4", rows=5, n=10007, k=2080, x="fp8", y="f32"),
        # a wide gate-and-up projection for a larger batch
        dict(name="w4_wide", op="w4", rows=64, n=16384, k=4096, x="bf16", y="bf16"),
        # the output head of a decode batch: the longest stream of weights
        dict(name="w4_head", op="w4", rows=16, n=131072, k=4096, x="bf16", y="f32"),
        # the answer of one token with twenty alternatives: one long row over the whole chip
        dict(name="logprobs_token", op="logprobs", rows=1, vocab=131072, kind="f32", given=1, top=20, masked=False, scale=1.0),
        # constrained sampling: most of the vocabulary masked, one row with nothing left, odd row starts, padding ids
        dict(name="logprobs_masked", op="logprobs", rows=37, vocab=50003, kind="bf16", given=3, top=8, masked=True, scale=1.25),
        # scoring a prompt
        dict(name="logprobs_prompt", op="logprobs", rows=2048, vocab=131072, kind="bf16", given=1, top=5, masked=False, scale=1.0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["join", "w4", "logprobs"])
    if op == "join":
        cols = _log_int(rng, 32, 8192)
        wire = rng.random() < 0.4
        cols = max(32, cols // 32 * 32) if wire else cols
        rows = _log_int(rng, 1, min(8192, 8192 * 4096 // cols))
        return dict(op=op, rows=rows, cols=cols, planes=rng.randint(1, 4), post=rng.random() < 0.5,
                    gate=rng.choice(["none", "row", "column", "full"]), wire=wire)
    if op == "w4":
        k = 32 * _log_int(rng, 1, 512)
        n = _log_int(rng, 16, min(131072, 131072 * 4096 // k))
        rows = _log_int(rng, 1, max(1, min(64, 16 * 131072 * 4096 // (n * k))))
        return dict(op=op, rows=rows, n=n, k=k, x=rng.choice(["bf16", "bf16", "fp8"]), y=rng.choice(["f32", "bf16"]))
    vocab = _log_int(rng, 64, 200000)
    rows = _log_int(rng, 1, min(2048, 2048 * 131072 // vocab // 2))
    return dict(op=op, rows=rows, vocab=vocab, kind=rng.choice(["f32", "bf16"]), given=rng.randint(1, 4), top=rng.randint(0, 32),
                masked=rng.random() < 0.4, scale=rng.choice([1.0, 0.7, 1.25]))


# ---- inputs ----------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"join": _prepare_join, "w4": _prepare_w4, "logprobs": _prepare_logprobs}[case["op"]](dict(case), g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_join(s, g):
    rows, cols = s["rows"], s["cols"]
    outlier = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.005, 20.0, 1.0)  # residual streams have a few loud channels
    s["h"] = _randn(g, rows, cols) * outlier
    s["planes_in"] = [(_randn(g, rows, cols) * 0.3).to(torch.bfloat16) for _ in range(s["planes"])]
    s["pre_w"] = 1.0 + 0.2 * _randn(g, cols)
    s["post_w"] = 0.5 + 0.1 * _randn(g, cols) if s["post"] else None
    shape = {"none": None, "row": (rows,), "column": (cols,), "full": (rows, cols)}[s["gate"]]
    s["gate_in"] = torch.sigmoid(_randn(g, *shape)) if shape else None
    s["branch_scale"] = 0.75
    s["h_out"] = torch.empty_like(s["h"])
    s["norm"] = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    if s["wire"]:  # rows of a request frame: payload, then scales, eight-byte aligned
        pitch = (cols + cols // WIRE_BLOCK + 7) // 8 * 8
        s["frame"] = torch.zeros(rows, pitch, dtype=torch.uint8, device="cuda")
        s["payload"] = s["frame"][:, :cols].view(torch.float8_e4m3fn)
        s["scales"] = s["frame"][:, cols:cols + cols // WIRE_BLOCK].view(torch.float8_e8m0fnu)
    if own:
        from mimo26f_afd_amd import coord
        pitch = s["frame"].shape[1] if s["wire"] else 0
        s["plan"] = coord.Join(cols, s["pre_w"].data_ptr(), post_weight=s["post_w"].data_ptr() if s["post"] else None,
                               planes=s["planes"], gate_cols={"none": 0, "row": 1}.get(s["gate"], cols),
                               gate_pitch={"row": 1, "full": cols}.get(s["gate"], 0), scale=s["branch_scale"], eps=EPS,
                               payload_pitch=pitch, scales_pitch=pitch)
    return s


def _prepare_w4(s, g):
    rows, n, k = s["rows"], s["n"], s["k"]
    s["w_payload"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s["w_scales"] = torch.randint(117, 121, (n, k // WIRE_BLOCK), generator=g, device="cuda", dtype=torch.uint8)
    empty = torch.rand(n, k // WIRE_BLOCK, generator=g, device="cuda") < 0.001  # groups of zeros carry the scale byte 0
    s["w_scales"].masked_fill_(empty, 0)
    s["w_payload"].view(n, k // WIRE_BLOCK, WIRE_BLOCK // 2).masked_fill_(empty[..., None], 0)
    x = _randn(g, rows, k)
    if s["x"] == "fp8":
        value, exponent = _wire(x)
        s["x_payload"], s["x_scales"] = value.to(torch.float8_e4m3fn).view(torch.uint8), exponent.to(torch.uint8)
    else:
        s["x_in"] = x.to(torch.bfloat16)
    s["out"] = torch.empty(rows, n, device="cuda", dtype=torch.float32 if s["y"] == "f32" else torch.bfloat16)
    if own:
        from mimo26f_afd_amd import coord
        s["weights"] = coord.Weights4(s["w_payload"].data_ptr(), s["w_scales"].data_ptr(), n, k)
    return s


def _prepare_logprobs(s, g):
    rows, vocab = s["rows"], s["vocab"]
    x = _randn(g, rows, vocab).mul_(2.5)
    loud = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
    x.scatter_add_(1, loud, 4.0 + 6.0 * torch.rand(rows, 12, generator=g, device="cuda"))
    if s["masked"]:
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < 0.9, -math.inf)
        if rows > 2:
            x[1] = -math.inf
    s["logits"] = x if s["kind"] == "f32" else x.to(torch.bfloat16)
    ids = torch.randint(0, vocab, (rows, s["given"]), generator=g, device="cuda", dtype=torch.int32)
    ids[:, 0] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.7, loud[:, 0], ids[:, 0])
    if rows > 4:
        ids[-1] = -1  # padding of a ragged batch: no token there
    s["ids"] = ids
    s["given_logprob"] = torch.empty(rows, s["given"], device="cuda")
    s["entropy"] = torch.empty(rows, device="cuda")
    s["top_ids"] = torch.empty(rows, s["top"], dtype=torch.int32, device="cuda")
    s["top_logprob"] = torch.empty(rows, s["top"], device="cuda")
    if own:
        from mimo26f_afd_amd import coord
        size = coord.token_logprobs_workspace(rows, vocab, s["top"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        s["workspace_bytes"] = size
    return s


# ---- one pass --------------------------------------------------------------------------------------

def run(s):
    return (_OWN if own else _PLAIN)[s["op"]](s)


def _own_join(s):
    s["plan"](s["rows"], s["h"].data_ptr(), [p.data_ptr() for p in s["planes_in"]], s["h_out"].data_ptr(), s["norm"].data_ptr(),
              gate=s["gate_in"].data_ptr() if s["gate_in"] is not None else None,
              payload=s["frame"].data_ptr() if s["wire"] else None,
              scales=s["frame"].data_ptr() + s["cols"] if s["wire"] else None)
    out = {"h": s["h_out"], "norm": s["norm"]}
    if s["wire"]:
        out.update(payload=s["payload"], scales=s["scales"])
    return out


def _own_w4(s):
    bf16 = s["y"] == "bf16"
    if s["x"] == "fp8":
        s["weights"].matvec_fp8(s["x_payload"].data_ptr(), s["x_scales"].data_ptr(), s["rows"], s["out"].data_ptr(), bf16)
    else:
        s["weights"].matvec(s["x_in"].data_ptr(), s["rows"], s["out"].data_ptr(), bf16)
    return s["out"]


def _own_logprobs(s):
    from mimo26f_afd_amd import coord
    coord.token_logprobs(s["logits"].data_ptr(), s["kind"] == "bf16", s["rows"], s["vocab"], s["vocab"], s["ids"].data_ptr(), s["given"],
                         s["given_logprob"].data_ptr(), s["entropy"].data_ptr(), s["top"], s["top_ids"].data_ptr(),
                         s["top_logprob"].data_ptr(), s["workspace"].data_ptr(), s["workspace_bytes"], scale=s["scale"])
    out = {"given": s["given_logprob"], "entropy": s["entropy"]}
    if s["top"]:
        out.update(top_ids=s["top_ids"], top=s["top_logprob"])
    return out


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _wire_exponent(x):
    """Scale byte of each block of 32: the smallest e with amax <= 448 * 2^e, plus 127, 0 for a block of zeros."""
    amax = x.unflatten(-1, (-1, WIRE_BLOCK)).abs().amax(-1)
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, (torch.where(m <= 0.875, e - 9, e - 8) + 127).clamp(0, 254), 0)


def _wire(x):
    """(values of the E4M3 codes, scale bytes): nearest code, halves away from zero, at most 448."""
    byte = _wire_exponent(x)
    y = x.unflatten(-1, (-1, WIRE_BLOCK)) * torch.exp2((127 - byte).float())[..., None]
    mag = y.abs().clamp(max=448.0)
    quantum = torch.exp2((torch.frexp(mag)[1] - 1).clamp(min=-6).float() - 3.0)
    value = torch.floor(mag / quantum + 0.5) * quantum
    return torch.copysign(value.clamp(max=448.0), y).flatten(-2), byte


def _plain_join(s):
    z = s["planes_in"][0].float()
    if s["planes"] > 1:
        z = torch.stack(s["planes_in"]).float().cumsum(0)[-1]
    if s["post"]:
        z = _rms(z, s["post_w"])
    if s["gate_in"] is not None:
        z = z * (s["gate_in"][:, None] if s["gate"] == "row" else s["gate_in"])
    h = s["h"] + s["branch_scale"] * z
    n = _rms(h, s["pre_w"])
    out = {"h": h, "norm": n.to(torch.bfloat16)}
    if s["wire"]:
        value, byte = _wire(n)
        out.update(payload=value.to(torch.float8_e4m3fn), scales=byte.to(torch.uint8).view(torch.float8_e8m0fnu))
    return out


def _plain_w4(s):
    n, k = s["n"], s["k"]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    codes = torch.stack([s["w_payload"] & 15, s["w_payload"] >> 4], -1).view(n, k // WIRE_BLOCK, WIRE_BLOCK)
    w = (table[codes.int()] * torch.exp2(s["w_scales"].float() - 127.0)[..., None]).view(n, k)
    if s["x"] == "fp8":
        x = s["x_payload"].view(torch.float8_e4m3fn).float().unflatten(-1, (-1, WIRE_BLOCK))
        x = (x * torch.exp2(s["x_scales"].float() - 127.0)[..., None]).flatten(-2)
    else:
        x = s["x_in"].float()
    y = x @ w.t()
    return y if s["y"] == "f32" else y.to(torch.bfloat16)


def _plain_logprobs(s):
    raw, vocab = s["logits"].float(), s["vocab"]
    x = raw * s["scale"]
    m = x.amax(-1, keepdim=True)
    empty = m == -math.inf
    d = x - torch.where(empty, 0.0, m)
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    log_z = torch.where(empty, 0.0, torch.log(z))
    mean = torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / torch.where(empty, 1.0, z)
    shift = torch.where(empty, 0.0, m) + log_z
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < vocab)
    given = torch.where(there, x.gather(1, ids.clamp(0, vocab - 1)) - shift, math.nan)
    out = {"given": given, "entropy": (log_z - mean)[:, 0]}
    if s["top"]:
        bits = (raw + 0.0).view(torch.int32)
        order = bits ^ ((bits >> 31) & 0x7FFFFFFF)  # signed integers in the order of the values
        place = vocab - 1 - torch.arange(vocab, device="cuda")
        key = (order.long() << 32) | place
        if s["top"] > vocab:
            raise ValueError("more alternatives than tokens")
        at = vocab - 1 - (torch.topk(key, s["top"], dim=-1).values & 0xFFFFFFFF)
        top = x.gather(1, at) - shift
        gone = top == -math.inf
        out.update(top_ids=torch.where(gone, -1, at).int(), top=top)
    return out


_OWN = {"join": _own_join, "w4": _own_w4, "logprobs": _own_logprobs}
_PLAIN = {"join": _plain_join, "w4": _plain_w4, "logprobs": _plain_logprobs}


# ---- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    if case["op"] == "join":
        rows, cols = case["rows"], case["cols"]
        gate = {"none": 0, "row": rows, "column": cols, "full": rows * cols}[case["gate"]]
        wire = cols + cols // WIRE_BLOCK if case["wire"] else 0
        return {"bytes": rows * (cols * (2 * case["planes"] + 4 + 4 + 2) + wire) + 4 * cols * (1 + case["post"]) + 4 * gate,
                "flops": rows * cols * (8 + case["planes"])}
    if case["op"] == "w4":
        rows, n, k = case["rows"], case["n"], case["k"]
        x = rows * (k + k // WIRE_BLOCK if case["x"] == "fp8" else 2 * k)
        return {"bytes": n * (k // 2 + k // WIRE_BLOCK) + x + rows * n * (4 if case["y"] == "f32" else 2), "flops": 2 * rows * n * k}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * (4 if case["kind"] == "f32" else 2) + 8 * case["given"] + 4 + 8 * case["top"]), "flops": 6 * rows * vocab}


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"join": _exact_join, "w4": _exact_w4, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_join(s):
    """h' = h + scale * gate * norm(sum of planes), then norm(h'); the wire codes as the numbers they round."""
    z = sum(p.double() for p in s["planes_in"])
    if s["post"]:
        z = z / (z.pow(2).sum(-1, keepdim=True) / s["cols"] + EPS).sqrt() * s["post_w"].double()
    if s["gate"] != "none":
        z = z * s["gate_in"].double().reshape((-1, 1) if s["gate"] == "row" else (-1, s["cols"]))
    h = s["h"].double() + s["branch_scale"] * z
    n = h / (h.pow(2).sum(-1, keepdim=True) / s["cols"] + EPS).sqrt() * s["pre_w"].double()
    out = {"h": h, "norm": n}
    if s["wire"]:
        blocks = n.reshape(s["rows"], -1, WIRE_BLOCK)
        amax = blocks.abs().max(-1).values
        e = torch.ceil(torch.log2(amax / 448.0)).clamp(-127, 127)
        out.update(payload=(blocks * torch.exp2(-e)[..., None]).reshape(s["rows"], -1), scales=torch.exp2(e))
    return out


def _exact_w4(s):
    """y = x W^T with W's E2M1 codes taken apart: sign, two exponent bits, one fraction bit."""
    n, k = s["n"], s["k"]
    p = s["w_payload"].reshape(n, k // 2, 1)
    code = torch.cat([p % 16, p // 16], -1).reshape(n, -1, WIRE_BLOCK)
    exponent, fraction = (code // 2) % 4, (code % 2).double()
    w = torch.where(exponent == 0, 0.5 * fraction, (1.0 + 0.5 * fraction) * torch.exp2(exponent.double() - 1.0))
    w = torch.where(code >= 8, -w, w)
    w = (w * torch.exp2(s["w_scales"].double() - 127.0).unsqueeze(-1)).reshape(n, k)
    if s["x"] == "fp8":
        x = s["x_payload"].view(torch.float8_e4m3fn).double() * torch.exp2(s["x_scales"].double() - 127.0).repeat_interleave(WIRE_BLOCK, -1)
    else:
        x = s["x_in"].double()
    return torch.mm(x, w.t())


def _exact_logprobs(s):
    """log softmax of the scaled logits at the given ids, its entropy, and its largest values."""
    out, rows = {"given": [], "entropy": [], "top": []}, s["rows"]
    for at in range(0, rows, 256):  # a slice of rows at a time: the intermediates are eight bytes a value
        x = s["logits"][at:at + 256].double() * s["scale"]
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        logp = torch.where(x == -math.inf, -math.inf, logp)
        p = torch.exp(logp)
        out["entropy"].append(-torch.where(p > 0, p * logp, 0.0).sum(-1))
        ids = s["ids"][at:at + 256].long()
        inside = (ids >= 0) & (ids < s["vocab"])
        got = torch.take_along_dim(logp, torch.where(inside, ids, 0), 1)
        out["given"].append(torch.where(inside, got, math.nan))
        out["top"].append(torch.sort(logp, -1, descending=True).values[:, :s["top"]])
    out = {k: torch.cat(v) for k, v in out.items()}
    if s["top"]:
        out["top_ids"] = None
    else:
        del out["top"]
    return out
