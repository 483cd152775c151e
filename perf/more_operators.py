"""What a batch whose sequences branch takes beside its forward passes: drawing each sequence's token from its own random number
and filters, and moving the rows of the generation state (and of the sampler's penalties) when sequences fork, end or make room.

A case is a dict of plain values.  Two operators; `kind`:

  draw     one token per row from `rows` rows of `vocab` logits (f32 or f16) with temperature, top-k, top-p and min-p of its own
           (`style`, below) and a given uniform random number (`hip.draw_tokens`); `shared`: all rows draw from one row of logits;
           `penalties`: repetition penalties are subtracted and brought up to date
  fork     in a pool of `rows` sequences, copies of the first `sources` ones in `moves` other places (`hip.copy_rows`, in place)
  compact  in a pool of `rows` sequences, `moves` live rows into the places of ended ones, as many other ended ones cleared (in place)
  gather   `moves` rows of a batch of `rows` into a narrower state of their own, every `fresh`th of them an empty one (0: none)

`run` computes the plain form, or calls the package where `own` is true.  listed() -> cases; draw(rng) -> one more case of the
same ranges; prepare(case, seed) -> what a program holds before the call; run(state) -> the outputs of one pass; exact(case, seed)
-> the same outputs from the definitions in 64 bits; work(case) -> bytes and operations that a pass cannot do without.
"""
import math

import torch

own = False

# layers, channels, heads of the package's presets
SHAPES = {"0.1B": (12, 768, 12), "1.5B": (24, 2048, 32), "7.2B": (32, 4096, 64)}
# temperature, top_k, top_p, min_p of one request.  "default": the engine's own options
STYLES = {"default": (1.0, 20, 0.3, 0.0), "chat": (0.8, 50, 0.9, 0.0), "nucleus": (1.0, 0, 0.95, 0.0), "min-p": (1.2, 0, 1.0, 0.05),
          "free": (1.0, 0, 1.0, 0.0), "greedy": (0.0, 0, 1.0, 0.0), "wide": (1.5, 1000, 0.99, 0.001)}
PRESENCE, FREQUENCY, DECAY = 2.0, 0.2, 0.996


def listed():
    return [
        # one user with the engine's default options: latency alone
        dict(name="draw 1 default", kind="draw", rows=1, vocab=65536, io="f32", style="default", shared=False, penalties=False),
        # eight answers to one prompt, the first token of each
        dict(name="draw 8 of one row min-p", kind="draw", rows=8, vocab=65536, io="f32", style="min-p", shared=True, penalties=False),
        # a full serving batch, every request with options of its own, repetition penalties on
        dict(name="draw 64 mixed penalties", kind="draw", rows=64, vocab=65536, io="f32", style="mixed", shared=False, penalties=True),
        # an odd vocabulary in half precision, where neighbours tie
        dict(name="draw 77x50277 f16 mixed", kind="draw", rows=77, vocab=50277, io="f16", style="mixed", shared=False, penalties=False),
        # a large batch that samples from the whole distribution
        dict(name="draw 256 free", kind="draw", rows=256, vocab=65536, io="f32", style="free", shared=False, penalties=False),
        # many rollouts at once with top-p alone: the sums over whole rows count
        dict(name="draw 512 nucleus", kind="draw", rows=512, vocab=65536, io="f32", style="nucleus", shared=False, penalties=False),
        # the smallest model's only sequence gets a copy
        dict(name="fork 0.1B 1", kind="fork", preset="0.1B", state="f32", rows=2, sources=1, moves=1, penalties=False),
        # sixteen answers to one prompt of the large model, penalties too
        dict(name="fork 7.2B f16 15", kind="fork", preset="7.2B", state="f16", rows=16, sources=1, moves=15, penalties=True),
        # a beam of three hypotheses that goes on as eleven
        dict(name="fork 1.5B 3 to 11", kind="fork", preset="1.5B", state="f32", rows=11, sources=3, moves=8, penalties=False),
        # a server's pool of sequences: ended ones make room
        dict(name="compact 7.2B 9 of 48", kind="compact", preset="7.2B", state="f32", rows=48, moves=9, penalties=True),
        # an odd number of live sequences goes on in a narrower batch with a few new ones
        dict(name="gather 1.5B f16 13 of 29", kind="gather", preset="1.5B", state="f16", rows=29, moves=13, fresh=5, penalties=False),
        # half of a full batch of the large model goes on: the largest call
        dict(name="gather 7.2B 32 of 64", kind="gather", preset="7.2B", state="f32", rows=64, moves=32, fresh=0, penalties=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["draw", "draw", "draw", "fork", "compact", "gather"])
    if kind == "draw":
        vocab = rng.choice([65536, 65536, _log_int(rng, 500, 131072)])
        penalties = rng.random() < 0.3
        rows = min(_log_int(rng, 1, 512), 512 * 65536 // vocab // (3 if penalties else 1))
        return dict(kind="draw", rows=rows, vocab=vocab, io=rng.choice(["f32", "f32", "f16"]), style=rng.choice(["mixed", "mixed", *STYLES]),
                    shared=rng.random() < 0.2, penalties=penalties)
    preset, state = rng.choice(list(SHAPES)), rng.choice(["f32", "f16"])
    rows = _log_int(rng, 4, 64)
    case = dict(kind=kind, preset=preset, state=state, rows=rows, penalties=rng.random() < 0.5)
    if kind == "fork":
        case["sources"] = rng.randint(1, max(1, rows // 4))
        case["moves"] = rng.randint(1, min(rows - case["sources"], 31))
    elif kind == "compact":
        case["moves"] = rng.randint(1, min(rows // 4, 16))
    else:
        case["moves"] = rng.randint(1, min(rows, 32))
        case["fresh"] = rng.choice([0, 0, 3, 5])
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _draw_inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    rows, V = case["rows"], case["vocab"]
    of = 1 if case["shared"] else rows
    # a broad floor and eight likely continuations per row, from no idea to nearly sure; one entry in fifty masked
    logits = torch.randn(of, V, generator=g, device="cuda").mul_(2.5).sub_(3.0)
    at = torch.randint(0, V, (of, 8), generator=g, device="cuda")
    logits.scatter_add_(1, at, rand(of, 8) * 10.0 + rand(of, 1) * 10.0)
    logits[:, torch.randint(0, V, (max(1, V // 50),), generator=g, device="cuda")] = float("-inf")
    names = list(STYLES) if case["style"] == "mixed" else [case["style"]]
    which = torch.randint(0, len(names), (rows,), generator=g, device="cuda")
    table = torch.tensor([STYLES[n] for n in names], device="cuda", dtype=torch.float32)[which]
    out = dict(logits=logits.to(torch.float16 if case["io"] == "f16" else torch.float32), uniform=rand(rows),
               temperature=table[:, 0].contiguous(), top_k=table[:, 1].int().contiguous(), top_p=table[:, 2].contiguous(),
               min_p=table[:, 3].contiguous(), source=torch.zeros(rows, dtype=torch.int32, device="cuda") if case["shared"] else None)
    if case["penalties"]:
        # a few hundred tokens of an answer so far
        p = torch.zeros(rows, V, device="cuda")
        said = torch.randint(0, V, (rows, 300), generator=g, device="cuda")
        said[:, :2] = at[torch.arange(rows, device="cuda") % of][:, :2]  # the likely ones among them
        out["penalties"] = p.scatter_reduce_(1, said, PRESENCE * DECAY ** (300.0 * rand(rows, 300)), "amax")
        new = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
        out.update(presence=new(PRESENCE), frequency=new(FREQUENCY), decay=new(DECAY))
    return out


def _tensors(case):
    """name -> (planes, bytes' shape of a row, type) of what a sequence keeps"""
    L, C, H = SHAPES[case["preset"]]
    out = {"shift": (2 * L, (C,), torch.float16), "wkv": (L, (H, 64, 64), torch.float32 if case["state"] == "f32" else torch.float16),
           "elapsed": (1, (), torch.int32)}
    if case["penalties"]:
        out["penalties"] = (1, (65536,), torch.float32)
    return out


def _moves(case, seed):
    """(destination, source) rows; source -1: cleared"""
    order = torch.randperm(case["rows"], generator=torch.Generator().manual_seed(seed)).tolist()
    n = case["moves"]
    if case["kind"] == "fork":
        sources, free = order[: case["sources"]], order[case["sources"]:]
        return [(d, sources[i % len(sources)]) for i, d in enumerate(free[:n])]
    if case["kind"] == "compact":
        ended = sorted(order[: 2 * n])
        live = sorted(order[2 * n:])[-n:]
        return list(zip(ended[:n], live)) + [(d, -1) for d in ended[n:]]
    keep = sorted(order[:n])
    return [(i, -1 if case["fresh"] and i % case["fresh"] == case["fresh"] - 1 else r) for i, r in enumerate(keep)]


def _state_inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    tensors = {}
    for name, (planes, row, dtype) in _tensors(case).items():
        shape = (planes, case["rows"], *row)
        if dtype == torch.int32:
            tensors[name] = torch.randint(0, 100000, shape, generator=g, device="cuda", dtype=dtype)
        else:
            tensors[name] = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    return tensors


def prepare(case, seed):
    if case["kind"] == "draw":
        state = dict(_draw_inputs(case, seed), case=case)
        if own:
            import numpy as np

            from rwkv_lightning_cuda_amd import hip

            rows = case["rows"]
            state["out"] = dict(token=torch.empty(rows, dtype=torch.int32, device="cuda"), logprob=torch.empty(rows, device="cuda"))
            if case["penalties"]:
                state["out"]["penalties"] = torch.empty_like(state["penalties"])
            state["workspace"] = hip.DeviceArray((hip.draw_tokens_workspace(rows, case["vocab"]),), np.uint8)
        return state
    state = dict(case=case, tensors=_state_inputs(case, seed), moves=_moves(case, seed))
    if case["kind"] == "gather":
        state["narrow"] = {k: torch.empty((t.shape[0], case["moves"], *t.shape[2:]), dtype=t.dtype, device="cuda") for k, t in state["tensors"].items()}
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _draw(s):
    case = s["case"]
    z = s["logits"].float()
    if s["source"] is not None:
        z = z[s["source"].long()]
    if case["penalties"]:
        z = z - s["penalties"]
    rows, V = z.shape
    # powers and sums in 64 bits: a draw next to a border goes by their last digits
    t = s["temperature"].double()[:, None]
    y = (z - z.amax(dim=1, keepdim=True)).double() * (math.log2(math.e) / torch.where(t > 0, t, 1.0))
    e = torch.where(y < -1000.0, 0.0, torch.exp2(y))
    # the order "larger first, equal ones by index": keys that hold the value's order above the index
    bits = (z + 0.0).view(torch.int32)
    key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) + torch.arange(V - 1, -1, -1, device=z.device)
    order = V - 1 - (torch.sort(key, dim=1, descending=True).values & 0xFFFFFFFF)
    before = torch.cumsum(e.gather(1, order), dim=1)
    top_p, min_p, top_k = s["top_p"].double()[:, None], s["min_p"].double()[:, None], s["top_k"].long()[:, None]
    everything = torch.full_like(top_k, V)
    n = torch.where(top_p < 1, (before < top_p * e.sum(dim=1, keepdim=True)).sum(dim=1, keepdim=True) + 1, everything)
    n = torch.minimum(n, torch.where(top_k > 0, top_k, everything))
    n = torch.minimum(n, torch.where(min_p > 0, (e >= min_p.clamp(max=1.0)).sum(dim=1, keepdim=True), everything))
    n = torch.where(t > 0, n.clamp(min=1), 1)
    kept = torch.zeros_like(e).scatter_(1, order, (torch.arange(V, device=z.device) < n).double()) * e
    upto = torch.cumsum(kept, dim=1)
    mass = upto[:, -1:]
    last = (V - 1 - (kept > 0).flip(1).int().argmax(dim=1, keepdim=True))
    token = torch.minimum((upto <= s["uniform"].double()[:, None] * mass).sum(dim=1, keepdim=True), last)
    # (through the others' share: near 0 where the token is nearly sure)
    own_e = e.gather(1, token)
    others = kept.scatter(1, token, 0.0).sum(dim=1, keepdim=True)
    out = {"token": token[:, 0].int(), "logprob": (-torch.log1p(others / own_e))[:, 0].float()}
    if case["penalties"]:
        p = s["penalties"]
        at = p.gather(1, token)
        add = torch.where(at == 0, s["presence"][:, None], s["frequency"][:, None])
        out["penalties"] = (p.double() * s["decay"].double()[:, None]).scatter_add_(1, token, add.double()).float()
    return out


def _plain_moves(s):
    kind = s["case"]["kind"]
    tensors = s["tensors"]
    to = torch.tensor([d for d, r in s["moves"] if r >= 0], device="cuda")
    rows = torch.tensor([r for d, r in s["moves"] if r >= 0], device="cuda")
    clear = torch.tensor([d for d, r in s["moves"] if r < 0], device="cuda", dtype=torch.long)
    target = s["narrow"] if kind == "gather" else tensors
    for name, t in target.items():
        t[:, to] = tensors[name][:, rows]
        if clear.numel():
            t[:, clear] = 0
    return target


def run(s):
    case = s["case"]
    if not own:
        return _draw(s) if case["kind"] == "draw" else _plain_moves(s)
    from rwkv_lightning_cuda_amd import hip

    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if case["kind"] == "draw":
        o = s["out"]
        hip.draw_tokens(case["rows"], case["vocab"], p(s["logits"]), p(s["uniform"]), p(o["token"]), s["workspace"], logprob=p(o["logprob"]),
                        temperature=p(s["temperature"]), top_k=p(s["top_k"]), top_p=p(s["top_p"]), min_p=p(s["min_p"]),
                        source=p(s["source"]), logit_rows=s["logits"].shape[0], penalties=p(s.get("penalties")), presence=p(s.get("presence")),
                        frequency=p(s.get("frequency")), decay=p(s.get("decay")), penalties_out=p(o.get("penalties")),
                        io=hip.IO_F16 if case["io"] == "f16" else hip.IO_F32)
        return o
    tensors = s["tensors"]
    target = s["narrow"] if case["kind"] == "gather" else tensors
    hip.copy_rows([(p(target[k]), p(t), t.shape[0], t[0, 0].numel() * t.element_size()) for k, t in tensors.items()],
                  case["moves"] if case["kind"] == "gather" else case["rows"], case["rows"], [d for d, _ in s["moves"]], [r for _, r in s["moves"]])
    return target


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] != "draw":
        old, out = _state_inputs(case, seed), {}
        for name, t in old.items():
            rows = list(t.unbind(1)) if case["kind"] != "gather" else [None] * case["moves"]
            for d, r in _moves(case, seed):
                rows[d] = t[:, r] if r >= 0 else torch.zeros_like(t[:, 0])
            out[name] = torch.stack(rows, dim=1)
        return out
    s = _draw_inputs(case, seed)
    tokens, logprobs = [], []
    for i in range(case["rows"]):
        z = s["logits"][0 if case["shared"] else i].float()
        if case["penalties"]:
            z = z - s["penalties"][i]
        z = z.double()
        temperature = s["temperature"][i].item()
        values, order = torch.sort(z, descending=True, stable=True)
        keep = 1
        if temperature > 0:
            p = torch.softmax(values / temperature, dim=0)
            keep = z.numel()
            if s["top_k"][i] > 0:
                keep = min(keep, s["top_k"][i].item())
            if s["top_p"][i] < 1:
                keep = min(keep, int((p.cumsum(0) < s["top_p"][i].double()).sum()) + 1)
            if s["min_p"][i] > 0:
                keep = min(keep, int((p >= s["min_p"][i].double() * p[0]).sum()))
        ids = order[:keep].sort().values
        logp = torch.log_softmax(z[ids] / (temperature if temperature > 0 else 1.0), dim=0)
        upto = logp.exp().cumsum(0)
        at = min(int(torch.searchsorted(upto, s["uniform"][i].double() * upto[-1], right=True)), keep - 1)
        tokens.append(ids[at].int())
        logprobs.append(logp[at])
    out = {"token": torch.stack(tokens), "logprob": torch.stack(logprobs)}
    if case["penalties"]:
        p = s["penalties"].double()
        at = out["token"].long()[:, None]
        add = torch.where(p.gather(1, at) == 0, s["presence"].double()[:, None], s["frequency"].double()[:, None])
        out["penalties"] = (p * s["decay"].double()[:, None]).scatter_add_(1, at, add)
    return out


def work(case):
    if case["kind"] == "draw":
        rows, V = case["rows"], case["vocab"]
        element = 2 if case["io"] == "f16" else 4
        # logits in; penalties in and out; parameters and results.  An entry: a difference, a power, comparisons, two sums
        return {"bytes": (1 if case["shared"] else rows) * V * element + (8 * rows * V if case["penalties"] else 0) + rows * 28, "flops": 20 * rows * V}
    row = sum(planes * math.prod(shape) * dtype.itemsize for planes, shape, dtype in _tensors(case).values())
    moves = _moves(case, 0)
    # each source row in once, each destination out once
    return {"bytes": row * (len({r for _, r in moves if r >= 0}) + len(moves)), "flops": 0}
