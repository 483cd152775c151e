"""What scoring a text takes behind the last layer: residual + norm with an 8-bit output, the vocabulary's product and the
log probabilities.

A case is a dict of plain values.  Three operators, by `kind`:

  norm      residual addition and LayerNorm or root-mean-square norm of `rows` rows of `width` fp16 values, in 8 bits with a
            scale per row (`hip.add_norm_q8`).  The 8-bit output comes back as the fp16 values it stands for.
  logprobs  from `rows` rows of `vocab` logits (f32 or f16): log probability and rank of each row's token, entropy, and the
            `top` most probable entries (`hip.token_logprobs`)
  head      the same, without the rank, for `rows` rows of hidden values in front of the vocabulary's matrix: the product and the
            log probabilities in one operator (`hip.linear_logprobs`).  `x` is fp16 or int8 with a scale per row, `weights` f16 or w8
            (int8 codes with an fp16 scale per vocabulary entry)

`run` computes the plain form, or calls the package where `own` is true.  listed() -> cases; draw(rng) -> one more case of the
same ranges; prepare(case, seed) -> what a program holds before the call; run(state) -> the outputs of one pass; exact(case, seed)
-> the same outputs from the definitions in 64 bits; work(case) -> bytes and operations that a pass cannot do without.
"""
import torch

own = False

EPS = 1e-5


def listed():
    return [
        # one token of the smallest model: latency alone
        dict(name="norm 1x768", kind="norm", norm="layer", rows=1, width=768, res=True),
        # a ragged prompt in a model with root-mean-square norms
        dict(name="norm rms 333x2048", kind="norm", norm="rms", rows=333, width=2048, res=True),
        # sixteen prompt chunks of the large model
        dict(name="norm 2048x4096", kind="norm", norm="layer", rows=2048, width=4096, res=True),
        # one reply with its five alternatives, after each sampled token
        dict(name="logprobs 1 top 5", kind="logprobs", rows=1, vocab=65536, io="f32", top=5),
        # a full serving batch that asks for as many alternatives as servers give
        dict(name="logprobs 64 top 20", kind="logprobs", rows=64, vocab=65536, io="f32", top=20),
        # an odd vocabulary in half precision, where neighbours tie
        dict(name="logprobs 77x50277 f16 top 3", kind="logprobs", rows=77, vocab=50277, io="f16", top=3),
        # every position of a batch of texts, likelihood and entropy only
        dict(name="logprobs 2048", kind="logprobs", rows=2048, vocab=65536, io="f32", top=0),
        # the smallest model's head for one position
        dict(name="head 1x768 f16", kind="head", rows=1, vocab=65536, width=768, x="f16", weights="f16", top=0),
        # the large model's head for one position: the weights' bytes count
        dict(name="head 1x4096 i8 top 5", kind="head", rows=1, vocab=65536, width=4096, x="i8", weights="w8", top=5),
        # an odd number of short texts, 8-bit weights under fp16 values
        dict(name="head 13x2048 w8", kind="head", rows=13, vocab=65536, width=2048, x="f16", weights="w8", top=0),
        # a ragged text in the middle model, unquantised
        dict(name="head 333x2048 f16", kind="head", rows=333, vocab=65536, width=2048, x="f16", weights="f16", top=0),
        # a batch of texts in the large model, 8 bits on both sides, with alternatives: the largest call
        dict(name="head 2048x4096 i8 top 5", kind="head", rows=2048, vocab=65536, width=4096, x="i8", weights="w8", top=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "logprobs", "logprobs", "head", "head"])
    if kind == "norm":
        width = rng.choice([768, 2048, 4096, 8 * _log_int(rng, 8, 1000)])
        return dict(kind="norm", norm=rng.choice(["layer", "rms"]), rows=_log_int(rng, 1, 2048), width=width, res=rng.random() < 0.7)
    if kind == "logprobs":
        vocab = rng.choice([65536, 65536, _log_int(rng, 500, 131072)])
        rows = min(_log_int(rng, 1, 2048), 2048 * 65536 // vocab)
        return dict(kind="logprobs", rows=rows, vocab=vocab, io=rng.choice(["f32", "f32", "f16"]), top=rng.choice([0, 1, 5, rng.randint(2, 20)]))
    vocab = rng.choice([65536, 65536, 32 * _log_int(rng, 20, 2048)])
    width = rng.choice([768, 2048, 4096, 256 * rng.randint(1, 15)])
    x, weights = rng.choice([("f16", "f16"), ("f16", "w8"), ("i8", "w8"), ("i8", "w8")])
    # (alternatives are whole numbers: only the products of whole numbers order the same however they are summed)
    top = rng.choice([0, 1, 5, rng.randint(2, 20)]) if x == "i8" else 0
    return dict(kind="head", rows=_log_int(rng, 1, 2000), vocab=vocab, width=width, x=x, weights=weights, top=top)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = case["rows"]
    if case["kind"] == "norm":
        C = case["width"]
        # a residual stream of a few standard deviations, some channels of it large as in trained models
        x = _randn(g, rows, C, std=2.0)
        x[:, :: max(1, C // 5)] *= 8.0
        return dict(x=x.half(), res=_randn(g, rows, C, dtype=torch.float16) if case["res"] else None,
                    w=_randn(g, C, std=0.1, mean=1.0, dtype=torch.float16),
                    b=_randn(g, C, std=0.1, dtype=torch.float16) if case["norm"] == "layer" else None)
    V = case["vocab"]
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if case["kind"] == "logprobs":
        # a broad floor, eight likely continuations per row, the given token mostly one of them, one entry in fifty masked
        logits = _randn(g, rows, V, std=2.5, mean=-3.0)
        at = torch.randint(0, V, (rows, 8), generator=g, device="cuda")
        logits.scatter_add_(1, at, torch.rand(rows, 8, generator=g, device="cuda") * 10.0 + 5.0)
        likely = torch.rand(rows, generator=g, device="cuda") < 0.7
        tokens = torch.where(likely, at[:, 0].int(), tokens)
        masked = torch.randint(0, V, (max(1, V // 50),), generator=g, device="cuda")
        logits[:, masked] = float("-inf")
        return dict(logits=logits.to(torch.float16 if case["io"] == "f16" else torch.float32), tokens=tokens)
    C = case["width"]
    out = dict(tokens=tokens)
    if case["weights"] == "f16":
        out["w"] = _randn(g, V, C, std=0.02, dtype=torch.float16)
        rows_of = out["w"][tokens.long()].float()
    else:
        codes = torch.randn(V, C, generator=g, device="cuda", dtype=torch.float16).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
        scale = ((torch.rand(V, generator=g, device="cuda") * 0.4 + 0.8) * (0.02 / 32.0)).half()
        out["w"], out["w_scale"] = codes, scale
        rows_of = codes[tokens.long()].float() * scale[tokens.long()].float()[:, None]
    # normalised hidden values that lean towards the token's own row: from no idea to nearly sure
    sure = torch.rand(rows, 1, generator=g, device="cuda") * 12.0
    x = _randn(g, rows, C) + sure * rows_of / rows_of.norm(dim=1, keepdim=True)
    if case["x"] == "f16":
        out["x"] = x.half()
    else:
        out["x_scale"] = x.abs().amax(dim=1) / 127.0
        out["x"] = (x / out["x_scale"][:, None]).round_().clamp_(-127, 127).to(torch.int8)
    return out


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        import numpy as np

        from rwkv_lightning_cuda_amd import hip

        rows = case["rows"]
        new = lambda *shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
        out = {}
        if case["kind"] == "norm":
            out["x_out"], out["values"] = new(*state["x"].shape, dtype=torch.float16), new(*state["x"].shape, dtype=torch.float16)
            out["scale"] = new(rows)
            state["q"] = new(*state["x"].shape, dtype=torch.int8)
        else:
            top = case["top"]
            out["logprob"], out["entropy"] = new(rows), new(rows)
            if case["kind"] == "logprobs":
                out["rank"] = new(rows, dtype=torch.int32)
                need = hip.token_logprobs_workspace(rows, case["vocab"], top)
            else:
                fmt = hip.FMT_F16 if case["weights"] == "f16" else hip.FMT_W8
                need = hip.linear_logprobs_workspace(fmt, rows, case["vocab"], case["width"], top, x_int8=case["x"] == "i8")
                # the matrix in the order that a model keeps for its products of several rows
                state["packed"] = torch.empty_like(state["w"])
                hip.pack_weights(fmt, case["vocab"], case["width"], state["w"].data_ptr(), state["packed"].data_ptr())
            if top:
                out["top_ids"], out["top_logprobs"] = new(rows, top, dtype=torch.int32), new(rows, top)
            state["workspace"] = hip.DeviceArray((need,), np.uint8) if need else None
        state["out"] = out
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _norm(s):
    x = s["x"].float()
    if s["res"] is not None:
        x = x + s["res"].float()
    c = x - x.mean(dim=1, keepdim=True) if s["case"]["norm"] == "layer" else x
    y = c * torch.rsqrt((c * c).mean(dim=1, keepdim=True) + EPS) * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    scale = y.abs().amax(dim=1) / 127.0
    q = (y / scale[:, None]).round()
    return {"x_out": x.half(), "values": (q * scale[:, None]).half(), "scale": scale}


def _ordered(logits, top):
    """The `top` largest entries of each row, equal ones by their index: keys that hold the value's order above the index."""
    bits = (logits + 0.0).view(torch.int32)
    key = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = (key.long() << 32) + torch.arange(logits.shape[1] - 1, -1, -1, device=logits.device)
    return logits.shape[1] - 1 - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)


def _of_logits(logits, tokens, top, rank):
    d = logits - logits.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    log_total = torch.log(total)
    at = tokens.long()[:, None]
    out = {"logprob": (d.gather(1, at) - log_total)[:, 0],
           "entropy": (log_total - torch.where(e > 0, d * e, 0.0).sum(dim=1, keepdim=True) / total)[:, 0]}
    if rank:
        own_logit = logits.gather(1, at)
        ahead = (logits > own_logit).sum(dim=1)
        index = torch.arange(logits.shape[1], device=logits.device)
        out["rank"] = (ahead + ((logits == own_logit) & (index < at)).sum(dim=1)).int()
    if top:
        ids = _ordered(logits, top)
        out["top_ids"], out["top_logprobs"] = ids.int(), d.gather(1, ids) - log_total
    return out


def _head(s):
    logits = s["x"].float() @ s["w"].float().t()
    if "w_scale" in s:
        logits = logits * s["w_scale"].float()
    if "x_scale" in s:
        logits = logits * s["x_scale"][:, None]
    return _of_logits(logits, s["tokens"], s["case"]["top"], False)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from rwkv_lightning_cuda_amd import hip

        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        o = s["out"]
        if kind == "norm":
            hip.add_norm_q8(case["rows"], case["width"], p(s["x"]), p(s["res"]), p(s["w"]), p(s["b"]), p(s["q"]), p(o["scale"]),
                            x_out=p(o["x_out"]), norm=hip.NORM_LAYER if case["norm"] == "layer" else hip.NORM_RMS, eps=EPS)
            # the values that the codes stand for, to compare: no part of the operator
            torch.mul(s["q"], o["scale"][:, None], out=o["values"])
        elif kind == "logprobs":
            hip.token_logprobs(case["rows"], case["vocab"], p(s["logits"]), p(s["tokens"]), s["workspace"], logprob=p(o["logprob"]),
                               entropy=p(o["entropy"]), rank=p(o["rank"]), top_n=case["top"], top_ids=p(o.get("top_ids")),
                               top_logprobs=p(o.get("top_logprobs")), io=hip.IO_F16 if case["io"] == "f16" else hip.IO_F32)
        else:
            hip.linear_logprobs(hip.FMT_F16 if case["weights"] == "f16" else hip.FMT_W8, case["rows"], case["vocab"], case["width"], p(s["x"]),
                                p(s["packed"]), p(s.get("w_scale")), p(s["tokens"]), s["workspace"], x_scale=p(s.get("x_scale")),
                                logprob=p(o["logprob"]), entropy=p(o["entropy"]), top_n=case["top"], top_ids=p(o.get("top_ids")),
                                top_logprobs=p(o.get("top_logprobs")))
        return o
    if kind == "norm":
        return _norm(s)
    if kind == "logprobs":
        return _of_logits(s["logits"].float(), s["tokens"], case["top"], True)
    return _head(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm":
        x = s["x"].double()
        if s["res"] is not None:
            x = x + s["res"].double()
        layer = case["norm"] == "layer"
        variance = x.var(dim=1, unbiased=False, keepdim=True) if layer else x.square().mean(dim=1, keepdim=True)
        y = (x - x.mean(dim=1, keepdim=True) if layer else x) / torch.sqrt(variance + EPS) * s["w"].double()
        if s["b"] is not None:
            y = y + s["b"].double()
        scale = y.abs().max(dim=1).values / 127.0
        return {"x_out": x, "values": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale}
    if case["kind"] == "logprobs":
        logits = s["logits"].double()
    else:
        x, w = s["x"].double(), s["w"].double()
        if "x_scale" in s:
            x = x * s["x_scale"].double()[:, None]
        if "w_scale" in s:
            w = w * s["w_scale"].double()[:, None]
        logits = torch.matmul(x, w.t().contiguous())
        del x, w
    lse = torch.logsumexp(logits, dim=1)
    logp = logits - lse[:, None]
    at = s["tokens"].long()[:, None]
    out = {"logprob": logp.gather(1, at)[:, 0], "entropy": torch.special.entr(logp.exp()).sum(dim=1)}
    if case["kind"] == "logprobs":
        out["rank"] = None
    if case["top"]:
        out["top_ids"] = None
        out["top_logprobs"] = logp.topk(case["top"], dim=1).values
    return out


def work(case):
    rows = case["rows"]
    if case["kind"] == "norm":
        n = rows * case["width"]
        # x and the residual in, the sum and the codes out, parameters, scales
        return {"bytes": n * (2 + (2 if case["res"] else 0) + 2 + 1) + case["width"] * (4 if case["norm"] == "layer" else 2) + rows * 4,
                "flops": 10 * n}
    V = case["vocab"]
    results = rows * (4 + 4 + 4 + 8 * case["top"])
    if case["kind"] == "logprobs":
        return {"bytes": rows * V * (2 if case["io"] == "f16" else 4) + results + rows * 4, "flops": 6 * rows * V}
    C = case["width"]
    return {"bytes": V * (2 * C if case["weights"] == "f16" else C + 2) + rows * (2 * C if case["x"] == "f16" else C + 4) + results,
            "flops": 2 * rows * V * C}
