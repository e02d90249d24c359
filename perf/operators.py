"""The operators around the LM head and the sampler, as measurable cases.

- Token log probabilities (`TokenLogprobs`): for each row of logits the log
  probabilities and ranks of given tokens, the normaliser, the entropy and the
  likeliest alternatives.
- Low-rank adapters (`LoraAdapters`): y_b += B_a (s_a A_a x_b) for the adapter
  a of each row b, beside the projection that all rows share.

Where `own` is false, `run` is the operator's plain form in torch.
"""
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NO_ADAPTER = -1


def _lp(rows, vocab, dtype, tokens, top, mask=0.0, softcap=0.0, temperature=False, pad=0):
    return {"kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "tokens": tokens,
            "top": top, "mask": mask, "softcap": softcap, "temperature": temperature, "pad": pad}


def _lora(batch, m, k, rank, adapters, weights, x, y, order, pad=0):
    return {"kind": "lora", "batch": batch, "m": m, "k": k, "rank": rank, "adapters": adapters,
            "weights": weights, "x": x, "y": y, "order": order, "pad": pad}


def listed():
    return [
        # one request on a 32k vocabulary that asks for the sampled token's and five alternatives' values: latency
        {"name": "logprobs_b1_v32000"} | _lp(1, 32000, "f32", 1, 5),
        # a decode batch (the headline's sizes) with the most alternatives that completion APIs offer
        {"name": "logprobs_b64_v128256"} | _lp(64, 128256, "f32", 1, 20),
        # structured output: about 3% of the tokens allowed, some rows with none, a temperature per row
        {"name": "logprobs_mask_b128_v128256"} | _lp(128, 128256, "f32", 1, 5, mask=0.03, temperature=True),
        # a large batch of bf16 logits
        {"name": "logprobs_bf16_b256_v151936"} | _lp(256, 151936, "bf16", 1, 8),
        # multiple choice: four candidate tokens per row, capped logits, rows of an odd size on 4-byte boundaries
        {"name": "logprobs_choice_b24_v50257"} | _lp(24, 50257, "f32", 4, 0, softcap=30.0, pad=6),
        # the largest batch and vocabulary of decode steps, with alternatives
        {"name": "logprobs_b512_v262144"} | _lp(512, 262144, "f32", 1, 10),
        # scoring the prompts of an evaluation: every position's own token, no alternatives
        {"name": "logprobs_prompt_b2048_v128256"} | _lp(2048, 128256, "bf16", 1, 0),
        # one request with its adapter: latency
        {"name": "lora_b1_m32000"} | _lora(1, 32000, 4096, 16, 1, "bf16", "f32", "f32", "mixed"),
        # a decode batch of many customers' requests, a few of them on the base model
        {"name": "lora_b64_m128256"} | _lora(64, 128256, 4096, 16, 16, "bf16", "f32", "f32", "mixed"),
        # nobody shares an adapter; 32-bit adapters of rank 8, sizes that divide nothing
        {"name": "lora_ragged_b24_m50257"} | _lora(24, 50257, 895, 8, 24, "f32", "f32", "f32", "each", pad=3),
        # few large adapters over a large batch, 16-bit throughout
        {"name": "lora_f16_b256_m151936"} | _lora(256, 151936, 2048, 64, 4, "f16", "bf16", "bf16", "mixed"),
        # prompts of different lengths, packed: long runs of rows on one adapter
        {"name": "lora_prompt_b1024_m128256"} | _lora(1024, 128256, 4096, 32, 8, "bf16", "f32", "f32", "packed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    vocab = _log_int(rng, 32000, 262144)
    if rng.random() < 0.5:
        vocab = max(32000, vocab // 128 * 128)  # half padded, half any size
    pad = rng.choice([0, 0, rng.randint(1, 64)])
    if rng.random() < 0.5:
        top = rng.choice([0, _log_int(rng, 1, 32)])
        tokens = rng.choice([1, 1, _log_int(rng, 2, 16)])
        rows = _log_int(rng, 1, 1024 if top == 0 and tokens == 1 else 256 if tokens <= 4 else 64)
        return _lp(rows, vocab, rng.choice(["f32", "bf16"]), tokens, top, rng.choice([0.0, 0.0, 0.03, 0.3]),
                   rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3, pad)
    batch = _log_int(rng, 1, 512)
    rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    adapters = min(_log_int(rng, 1, 64), 1024 // rank, max(1, 2 * batch))
    return _lora(batch, min(vocab, 151936), _log_int(rng, 896, 8192), rank, adapters,
                 rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["f32", "bf16"]),
                 rng.choice(["f32", "f32", "bf16"]), rng.choice(["mixed", "packed"]), pad)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _logprobs_inputs(case, seed):
    """Logits: N(0, 3) plus -1.1 ln(rank) over a permutation of the vocabulary (tokens are about
    as frequent in one row as in the next); a spread of 30 and more from likely to unlikely."""
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    prior = -1.1 * torch.log(_rand(g, vocab).argsort().float() + 1.0)
    logits = torch.empty(rows, vocab + case["pad"], device="cuda")
    logits.normal_(generator=g)
    logits.mul_(3.0)
    logits[:, :vocab] += prior
    logits = logits.to(DTYPES[case["dtype"]])[:, :vocab]
    # three rows in four hold their likeliest token among the given ones, as sampled tokens mostly are
    tokens = (_rand(g, rows, case["tokens"]) * vocab).int().clamp_(max=vocab - 1)
    likely = logits.argmax(dim=1).int()
    tokens[:, 0] = torch.where(_rand(g, rows) < 0.75, likely, tokens[:, 0])
    s = {"logits": logits, "tokens": tokens, "mask": None, "temperatures": None}
    if case["mask"]:
        words = (vocab + 31) // 32
        bits = _rand(g, rows, words * 32) < case["mask"]
        bits[:, vocab:] = False
        bits[rows // 3 + 1::61] = False  # rows whose grammar allows nothing
        bits[rows // 2::4] &= bits[rows // 2::4].int().cumsum(dim=1) <= 3  # and rows with three tokens at most
        weight = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device="cuda")
        s["mask"] = (bits.view(rows, words, 32) * weight).sum(dim=2).int()
    if case["temperature"]:
        s["temperatures"] = 0.5 + _rand(g, rows)
    return s


def _lora_inputs(case, seed):
    g = _gen(seed)
    batch, m, k, rank, n = case["batch"], case["m"], case["k"], case["rank"], case["adapters"]
    wt = DTYPES[case["weights"]]
    a = torch.empty(n, rank, k, dtype=wt, device="cuda")
    b = torch.empty(n, m, rank, dtype=wt, device="cuda")
    ranks = []
    for i in range(n):  # one adapter in three has half the rank; the rest of its slot is zero
        r = max(1, rank // 2) if i % 3 == 2 else rank
        ranks.append(r)
        a[i] = _randn(g, rank, k) / math.sqrt(k)
        b[i] = _randn(g, m, rank) * 0.1
        a[i, r:] = 0
        b[i, :, r:] = 0
    scales = 0.5 + 1.5 * _rand(g, n)
    ids = (_rand(g, batch) * n).int().clamp_(max=n - 1)
    if case["order"] == "each":
        ids = _rand(g, n).argsort()[:batch]
    elif case["order"] == "packed":
        ids = ids.sort().values
    elif batch > 8:
        ids = torch.where(_rand(g, batch) < 0.1, NO_ADAPTER, ids)  # requests on the base model
    x = (_randn(g, batch, k + case["pad"]) * 1.5).to(DTYPES[case["x"]])[:, :k]
    y = (_randn(g, batch, m + case["pad"]) * 3.0).to(DTYPES[case["y"]])[:, :m]
    return {"a": a, "b": b, "ranks": ranks, "scales": scales, "ids": ids.int(), "x": x, "y": y}


def prepare(case, seed):
    if case["kind"] == "logprobs":
        s = _logprobs_inputs(case, seed)
        s |= {"kind": "logprobs", "top": case["top"], "softcap": case["softcap"]}
    else:
        s = _lora_inputs(case, seed)
        s["kind"] = "lora"
    if own:
        package = str(ROOT / "oxide-tech-llm-engine_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from oxide_sampler import LoraAdapters, TokenLogprobs
        if case["kind"] == "logprobs":
            # a decode loop's buffers stay where they are: the call is described once
            s["handle"] = TokenLogprobs()
            s["call"], s["out"] = s["handle"].descriptor(
                s["logits"], s["tokens"], top=s["top"], mask=s["mask"], temperatures=s["temperatures"],
                softcap=s["softcap"])
        else:
            # the table that a server loads its adapters into
            s["handle"] = LoraAdapters(case["m"], case["k"], max_adapters=case["adapters"], max_rank=case["rank"],
                                       max_batch=case["batch"], dtype=DTYPES[case["weights"]])
            for i, (r, scale) in enumerate(zip(s["ranks"], s["scales"].tolist())):
                s["handle"].load(i, s["a"][i, :r], s["b"][i, :, :r], scale)
            s["call"] = s["handle"].descriptor(s["y"], s["x"], s["ids"])
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    if own:
        state["handle"].launch(state["call"])
        return {"y": state["y"]} if state["kind"] == "lora" else state["out"]
    return (_plain_lora if state["kind"] == "lora" else _plain_logprobs)(state)


def _allowed(mask, vocab):
    i = torch.arange(vocab, device=mask.device)
    return (mask[:, i >> 5] >> (i & 31)) & 1 != 0


def _plain_logprobs(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    absent = torch.isnan(x) | (x == -math.inf)
    if s["mask"] is not None:
        absent |= ~_allowed(s["mask"], vocab)
    x = torch.where(absent, -math.inf, x)
    z = s["softcap"] * torch.tanh(x / s["softcap"]) if s["softcap"] else x
    if s["temperatures"] is not None:
        z = z / s["temperatures"][:, None]
    z = torch.where(absent, -math.inf, z)
    best = z.amax(dim=1, keepdim=True)
    empty = best == -math.inf
    d = z - torch.where(empty, 0.0, best)
    e = torch.exp(d)
    total = torch.where(empty, 1.0, e.sum(dim=1, keepdim=True))
    shift = torch.log(total)
    token = s["tokens"].long()
    value = x.gather(1, token)[:, :, None]
    before = torch.arange(vocab, device=x.device) < token[:, :, None]
    rank = 1 + ((x[:, None, :] > value) | ((x[:, None, :] == value) & before)).sum(dim=2)
    out = {
        "logprobs": d.gather(1, token) - shift,
        "ranks": torch.where(value[:, :, 0] == -math.inf, 0, rank).int(),
        "logsumexp": (best + shift)[:, 0],
        "entropy": (shift - torch.where(e > 0, d * e, 0.0).sum(dim=1, keepdim=True) / total)[:, 0],
        "status": empty[:, 0].int(),
    }
    if s["top"]:
        # one whole number per logit: its value's order, then the lower id
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = (order << 32) - torch.arange(vocab, device=x.device)
        best_ids = key.topk(s["top"], dim=1).indices
        gone = absent.gather(1, best_ids)
        out["top_ids"] = torch.where(gone, -1, best_ids).int()
        out["top_logprobs"] = d.gather(1, best_ids) - shift
    return out


def _plain_lora(s):
    n, rank, k = s["a"].shape
    batch, m = s["y"].shape
    v = s["x"].float() @ s["a"].float().reshape(n * rank, k).T
    mine = s["ids"][:, None] == torch.arange(n, device=v.device)
    v = v.view(batch, n, rank) * (mine * s["scales"])[:, :, None]
    b = s["b"].float().transpose(1, 2).reshape(n * rank, m)
    s["y"].copy_(s["y"].float() + v.view(batch, n * rank) @ b)
    return {"y": s["y"]}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        read = rows * vocab * size + (rows * ((vocab + 31) // 32) * 4 if case["mask"] else 0) + rows * case["tokens"] * 4
        write = rows * (8 * case["tokens"] + 8 * case["top"] + 12)
        return {"bytes": read + write, "flops": 5 * rows * vocab}
    size = {"f32": 4, "bf16": 2, "f16": 2}
    batch, m, k, n = case["batch"], case["m"], case["k"], case["adapters"]
    rank = sum(max(1, case["rank"] // 2) if i % 3 == 2 else case["rank"] for i in range(n)) / n
    rows = 0.9 * batch if case["order"] == "mixed" and batch > 8 else batch  # the others are left alone
    used = min(n, rows) if case["order"] == "each" else n * (1 - (1 - 1 / n) ** rows)  # adapters that some row has
    weights = used * rank * (m + k) * size[case["weights"]]
    return {"bytes": weights + rows * (k * size[case["x"]] + 2 * m * size[case["y"]]),
            "flops": 2 * rows * rank * (m + k)}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    return (_exact_lora if case["kind"] == "lora" else _exact_logprobs)(case, seed)


def _exact_logprobs(case, seed):
    s = _logprobs_inputs(case, seed)
    out = []
    for r in range(0, case["rows"], 128):
        z = s["logits"][r:r + 128].double()
        if case["softcap"]:
            z = (z / case["softcap"]).tanh() * case["softcap"]
        if case["temperature"]:
            z = z / s["temperatures"][r:r + 128, None].double()
        if case["mask"]:
            words = s["mask"][r:r + 128, :, None]
            bit = words.bitwise_right_shift(torch.arange(32, dtype=torch.int32, device=z.device)).bitwise_and(1)
            z.masked_fill_(bit.flatten(1)[:, :case["vocab"]] == 0, -math.inf)
        some = (z > -math.inf).any(dim=1)
        lse = torch.logsumexp(z, dim=1)
        lp = z - torch.where(some, lse, 0.0)[:, None]
        p = lp.exp()
        tokens = s["tokens"][r:r + 128].long()
        part = {"logprobs": lp.gather(1, tokens), "logsumexp": lse, "entropy": -torch.special.xlogy(p, p).sum(dim=1)}
        if case["top"]:
            part["top_logprobs"] = lp.topk(case["top"], dim=1).values
        out.append(part)
    whole = {name: torch.cat([part[name] for part in out]) for name in out[0]}
    return whole | {"ranks": None, "status": None} | ({"top_ids": None} if case["top"] else {})


def _exact_lora(case, seed):
    s = _lora_inputs(case, seed)
    y = s["y"].double()
    for i, r in enumerate(s["ranks"]):
        rows = (s["ids"] == i).nonzero()[:, 0]
        if len(rows):
            v = s["x"][rows].double() @ s["a"][i, :r].double().T
            y[rows] += (v * s["scales"][i].double()) @ s["b"][i, :, :r].double().T
    return {"y": y}
