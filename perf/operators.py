"""The paged key/value cache operators, as they are measured: the cases, their plain forms and their exact values.

Three operators share one pool of cache pages. A pool is a pair of [pages, kv_heads, page_size, head_dim] bf16
tensors; row s of a page table names the pages of sequence s in order, so position p of sequence s lives in row
p % page_size of page table[s, p // page_size]:

* write:  QKV projection rows -> per-head q/k RMSNorm, rotate-half RoPE, queries out, K/V into their pages;
* decode: one new token per sequence attends to the sequence's keys 0 .. position;
* prompt: packed prompts of different lengths attend causally to their own sequence's pages (those written
  for the prompt itself and those that were cached before it).
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
BF16 = torch.bfloat16
EPS = 1e-6
# (query heads, key/value heads, head dim): the talker and the code predictor (16, 8, 128) and the codec's
# transformer (8, 8, 64) of this repository, then generic grouped layouts.
HEADS = ((16, 8, 128), (8, 8, 64), (32, 8, 128), (12, 4, 64), (14, 2, 64), (8, 1, 128), (6, 6, 128), (16, 1, 128))
PAGES = (16, 32, 64, 128, 256)


def listed():
    return [
        # one new token of one request: the latency of the smallest decode step
        dict(name="write-step-1", op="write", q=16, kv=8, d=128, page=16, count=1, lo=300, hi=300, new=1, norm=True,
             view=False, lens=1),
        # a decode step at the serving concurrency, contexts as the talker sees them
        dict(name="write-step-64", op="write", q=16, kv=8, d=128, page=64, count=64, lo=64, hi=1024, new=1, norm=True,
             view=False, lens=2),
        # an admission of sixteen prompts packed end to end
        dict(name="write-prompts-16", op="write", q=16, kv=8, d=128, page=32, count=16, lo=40, hi=400, new=0,
             norm=True, view=False, lens=3),
        # thousands of rows without head norms, read from the columns of a wider buffer
        dict(name="write-codec-rows", op="write", q=8, kv=8, d=64, page=128, count=11, lo=500, hi=1999, new=0,
             norm=False, view=True, lens=4),
        # one request early in its answer
        dict(name="decode-1", op="decode", q=16, kv=8, d=128, page=16, count=1, lo=97, hi=97, view=False, lens=5),
        # the serving concurrency with ragged contexts
        dict(name="decode-64", op="decode", q=16, kv=8, d=128, page=64, count=64, lo=64, hi=2048, view=False, lens=6),
        # a few requests with very long contexts
        dict(name="decode-long", op="decode", q=32, kv=8, d=128, page=128, count=3, lo=20000, hi=65535, view=True,
             lens=7),
        # a large batch over small pages
        dict(name="decode-256", op="decode", q=16, kv=8, d=128, page=16, count=256, lo=1, hi=4096, view=False, lens=8),
        # one short prompt
        dict(name="prompt-1", op="prompt", q=8, kv=8, d=64, page=16, count=1, lo=13, hi=13, clo=0, chi=0, view=False,
             lens=9),
        # an admission of sixteen prompts
        dict(name="prompt-16", op="prompt", q=16, kv=8, d=128, page=32, count=16, lo=40, hi=400, clo=0, chi=0,
             view=False, lens=10),
        # chunks of prompts whose beginnings are cached already
        dict(name="prompt-chunks", op="prompt", q=16, kv=8, d=128, page=256, count=4, lo=100, hi=700, clo=2000,
             chi=8000, view=True, lens=11),
        # one long prompt
        dict(name="prompt-long", op="prompt", q=32, kv=8, d=128, page=64, count=1, lo=8191, hi=8191, clo=0, chi=0,
             view=False, lens=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        q, kv, d = rng.choice(HEADS)
        c = dict(op=rng.choice(("write", "decode", "prompt")), q=q, kv=kv, d=d, page=rng.choice(PAGES),
                 view=rng.random() < 0.3, lens=rng.randrange(1 << 20))
        if c["op"] == "write":
            c["new"] = rng.choice((0, 1))
            c["norm"] = rng.random() < 0.7
            c["count"] = _log(rng, 1, 256) if c["new"] else _log(rng, 1, 32)
            c["hi"] = _log(rng, 1, 4096)
        elif c["op"] == "decode":
            c["count"], c["hi"] = _log(rng, 1, 256), _log(rng, 1, 65536)
        else:
            c["count"], c["hi"], c["chi"] = _log(rng, 1, 32), _log(rng, 1, 8192), rng.choice((0, _log(rng, 1, 16384)))
            c["clo"] = rng.randint(0, c["chi"])
        c["lo"] = rng.randint(1, c["hi"])
        # the ends of a batch of 256 rows, or the largest listed case of the operator
        top = dict(listed()[7], lo=2048) if c["op"] == "decode" else [t for t in listed() if t["op"] == c["op"]][-1]
        if _cost(c) <= _cost(top) and _padded(c) <= _padded(top):
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 250)


def _padded(c):
    """The elements that the plain form works on where every sequence is as long as the longest."""
    hi = c["hi"]
    if c["op"] == "write":
        return c["count"] * (1 if c["new"] else hi) * (c["q"] + 2 * c["kv"]) * c["d"]
    if c["op"] == "decode":
        return c["count"] * hi * c["kv"] * c["d"]
    return c["count"] * c["q"] * hi * (hi + c["chi"])


def _lengths(c):
    """The lengths of the case's sequences (fixed by the case, not by the seed of its values)."""
    r = random.Random(c["lens"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["count"])], \
           [r.randint(c.get("clo", 0), c.get("chi", 0)) for _ in range(c["count"])]


def work(c):
    n, cached = _lengths(c)
    q, kv, d = c["q"], c["kv"], c["d"]
    if c["op"] == "write":
        rows = len(n) if c["new"] else sum(n)
        # qkv in, the cos and sin rows, queries out, K and V out, positions
        return {"bytes": rows * (2 * (q + 2 * kv) * d * 2 + 2 * d * 2 + 24), "flops": rows * (q + kv) * d * 8}
    if c["op"] == "decode":
        keys = sum(n)
        return {"bytes": keys * kv * d * 4 + len(n) * (2 * q * d * 2 + 8), "flops": keys * q * d * 4}
    rows, keys = sum(n), sum(a + b for a, b in zip(n, cached))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, cached))
    return {"bytes": 2 * rows * q * d * 2 + keys * kv * d * 4, "flops": pairs * q * d * 4}


def _table(lengths, page, gen):
    """A pool's page count and the page table: pages handed out in a shuffled order, unused entries -1."""
    need = [-(-n // page) for n in lengths]
    total = sum(need)
    order = torch.randperm(total, generator=gen, dtype=torch.int32, device=DEVICE)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
    need_t = torch.tensor(need, device=DEVICE)
    column = torch.arange(max(need), device=DEVICE)
    at = (first[:, None] + column).clamp(max=total - 1)
    return total, torch.where(column < need_t[:, None], order[at], -1).to(torch.int32).contiguous()


def _rows(shape, view, gen):
    """bf16 normal rows; with `view` the leading columns of rows that are wider by 64."""
    rows, width = shape[0], math.prod(shape[1:])
    full = torch.randn(rows, width + (64 if view else 0), generator=gen, device=DEVICE).to(BF16)
    return full[:, :width].unflatten(1, shape[1:]) if len(shape) > 2 else full[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    n, cached = _lengths(case)
    q, kv, d, page = case["q"], case["kv"], case["d"], case["page"]
    lengths = [a + b for a, b in zip(n, cached)]
    pages, table = _table(lengths, page, gen)
    keys = torch.randn(pages, kv, page, d, generator=gen, device=DEVICE, dtype=BF16)
    values = torch.randn(pages, kv, page, d, generator=gen, device=DEVICE, dtype=BF16)
    s = dict(op=case["op"], q=q, kv=kv, d=d, keys=keys, values=values, table=table)
    if case["op"] == "write":
        if case["new"]:  # one row per sequence, at its last position
            rows = len(n)
            at = torch.tensor(n, device=DEVICE) - 1
            s["sequences"] = None
        else:            # every position of every sequence, packed end to end
            rows = sum(n)
            at = torch.cat([torch.arange(m, device=DEVICE) for m in n])
            s["sequences"] = torch.repeat_interleave(torch.arange(len(n), device=DEVICE), torch.tensor(n, device=DEVICE))
        span = max(n) + 8
        freq = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEVICE) / d)
        angle = torch.arange(span, dtype=torch.float64, device=DEVICE)[:, None] * freq
        s["cos"], s["sin"] = (f(torch.cat((angle, angle), 1)).to(BF16) for f in (torch.cos, torch.sin))
        s["qkv"] = _rows((rows, (q + 2 * kv) * d), case["view"], gen)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.1 * torch.randn(d, generator=gen, device=DEVICE)).to(BF16) for _ in "qk")
        s["cache_positions"], s["rotary_positions"] = at, at + seed % 8
        s["query"] = torch.zeros(rows, q, d, dtype=BF16, device=DEVICE)
    elif case["op"] == "decode":
        s["query"] = _rows((len(n), q, d), case["view"], gen)
        s["positions"] = torch.tensor(n, device=DEVICE) - 1
        s["out"] = torch.zeros(len(n), q, d, dtype=BF16, device=DEVICE)
        s["context"] = max(n)
    else:
        s["query"] = _rows((sum(n), q, d), case["view"], gen)
        s["row_offsets"] = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], device=DEVICE)
        s["start_positions"] = torch.tensor(cached, device=DEVICE)
        s["out"] = torch.zeros(sum(n), q, d, dtype=BF16, device=DEVICE)
        s["longest"], s["context"] = max(n), max(lengths)
    return s


_ops = None


def _framework():
    global _ops
    if _ops is None:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "qwen3-tts-rsi-engine_b200"))
        from qwen3_tts_b200 import ops
        _ops = ops
    return _ops


def run(s):
    if own:
        return _run_own(s)
    return {"write": _plain_write, "decode": _plain_decode, "prompt": _plain_prompt}[s["op"]](s)


def _run_own(s):
    ops = _ops or _framework()
    if s["op"] == "write":
        query = ops.paged_qk_norm_rope_kv(s["qkv"], s["q_norm"], s["k_norm"], EPS, s["cos"], s["sin"],
                                          s["rotary_positions"], s["cache_positions"], s["table"], s["keys"],
                                          s["values"], q_heads=s["q"], kv_heads=s["kv"], head_dim=s["d"],
                                          sequences=s["sequences"], query_out=s["query"])
        return [query, s["keys"], s["values"]]
    if s["op"] == "decode":
        return ops.paged_decode_attention(s["query"], s["keys"], s["values"], s["table"], s["positions"],
                                          context=s["context"], out=s["out"])
    return ops.paged_prefill_attention(s["query"], s["keys"], s["values"], s["table"], s["row_offsets"],
                                       s["start_positions"], out=s["out"])


# ------------------------------------------------------------------ plain forms
def _turn(x, weight, cos, sin):
    """Head norm (where there is a weight) and rotate-half RoPE of [rows, heads, dim] in 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin


def _plain_write(s):
    q, kv, d = s["q"], s["kv"], s["d"]
    rows = s["qkv"].unflatten(1, (q + 2 * kv, d))
    cos, sin = (t[s["rotary_positions"]].float()[:, None] for t in (s["cos"], s["sin"]))
    s["query"].copy_(_turn(rows[:, :q], s["q_norm"], cos, sin))
    page = s["keys"].shape[2]
    at = s["cache_positions"]
    sequences = torch.arange(len(at), device=at.device) if s["sequences"] is None else s["sequences"]
    pages = s["table"][sequences, at // page].long()
    s["keys"][pages, :, at % page] = _turn(rows[:, q:q + kv], s["k_norm"], cos, sin).to(BF16)
    s["values"][pages, :, at % page] = rows[:, q + kv:]
    return [s["query"], s["keys"], s["values"]]


def _gather(pool, table, context):
    """[sequences, kv_heads, context, dim] in 32 bits of the pages that a table names."""
    page = pool.shape[2]
    x = pool[table[:, :-(-context // page)].clamp(min=0).long()].float()
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :context]


def _softmax_product(scores, seen, values):
    scores = scores.masked_fill_(~seen, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    return scores @ values / scores.sum(-1, keepdim=True)


def _plain_decode(s):
    rows, q, d = s["query"].shape
    keys, values = (_gather(s[k], s["table"], s["context"]) for k in ("keys", "values"))
    seen = torch.arange(s["context"], device=keys.device) <= s["positions"][:, None]
    query = s["query"].float().unflatten(1, (s["kv"], -1)) * d ** -0.5
    s["out"].copy_(_softmax_product(query @ keys.mT, seen[:, None, None], values).flatten(1, 2))
    return s["out"]


def _plain_prompt(s):
    rows, q, d = s["query"].shape
    kv, longest = s["kv"], s["longest"]
    offsets, start = s["row_offsets"], s["start_positions"]
    keys, values = (_gather(s[k], s["table"], s["context"]) for k in ("keys", "values"))
    step = torch.arange(longest, device=keys.device)
    row = (offsets[:-1, None] + step).clamp(max=rows - 1)                       # [sequences, longest]
    query = s["query"][row].float().unflatten(2, (kv, -1)) * d ** -0.5          # [sequences, longest, kv, group, d]
    query = query.permute(0, 2, 3, 1, 4).flatten(2, 3)
    seen = torch.arange(s["context"], device=keys.device) <= (start[:, None] + step)[:, :, None]
    out = _softmax_product(query @ keys.mT, seen[:, None].repeat(1, 1, q // kv, 1), values)
    out = out.unflatten(2, (q // kv, longest))                                  # [sequences, kv, group, longest, d]
    index = torch.arange(rows, device=keys.device)
    sequence = torch.searchsorted(offsets, index, right=True) - 1
    s["out"].copy_(out[sequence, :, :, index - offsets[sequence]].flatten(1, 2))
    return s["out"]


# ------------------------------------------------------------------ exact values, in 64 bits
def exact(case, seed):
    def write(s):
        q, kv, d = s["q"], s["kv"], s["d"]
        if s["keys"].numel() > 1 << 28:
            return None
        x = s["qkv"].double().reshape(-1, q + 2 * kv, d)
        c, n = s["cos"].double()[s["rotary_positions"]], s["sin"].double()[s["rotary_positions"]]
        partner = torch.tensor([(i + d // 2) % d for i in range(d)], device=x.device)
        sign = torch.tensor([-1.0 if i < d // 2 else 1.0 for i in range(d)], dtype=torch.float64, device=x.device)

        def turned(h, weight):
            y = h
            if weight is not None:
                y = weight.double() * (h / torch.sqrt(torch.sum(h ** 2, -1, keepdim=True) / d + EPS))
            return torch.einsum("rhd,rd->rhd", y, c) + torch.einsum("rhd,rd->rhd", y[..., partner] * sign, n)

        keys, values = s["keys"].double(), s["values"].double()
        page = keys.shape[2]
        at = s["cache_positions"]
        k, v = turned(x[:, q:q + kv], s["k_norm"]), x[:, q + kv:]
        seq = s["sequences"] if s["sequences"] is not None else torch.arange(at.numel(), device=at.device)
        flat = s["table"].long().gather(0, seq[:, None].expand(-1, s["table"].shape[1])).gather(1, (at // page)[:, None])[:, 0]
        for h in range(kv):
            keys[flat, h, at % page] = k[:, h]
            values[flat, h, at % page] = v[:, h]
        return [turned(x[:, :q], s["q_norm"]), keys, values]

    def sequence(pool, table, length, head):
        """[length, dim] in 64 bits: one head of one sequence, page after page."""
        page = pool.shape[2]
        names = table[:-(-length // page)].long()
        return pool[:, head].index_select(0, names).reshape(-1, pool.shape[-1])[:length].double()

    def decode(s):
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
        group = s["q"] // s["kv"]
        if s["out"].shape[0] * s["kv"] > 4096:
            return None
        for r, p in enumerate(s["positions"].tolist()):
            for h in range(s["kv"]):
                k, v = (sequence(s[t], s["table"][r], p + 1, h) for t in ("keys", "values"))
                logits = torch.mv(k, s["query"][r, h * group].double()) if group == 1 else \
                    torch.mm(s["query"][r, h * group:(h + 1) * group].double(), k.t())
                weights = torch.softmax(logits / math.sqrt(s["d"]), -1)
                out[r, h * group:(h + 1) * group] = weights.reshape(-1, p + 1) @ v
        return out

    def prompt(s):
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
        group = s["q"] // s["kv"]
        offsets, start = s["row_offsets"].tolist(), s["start_positions"].tolist()
        for i, first in enumerate(start):
            lo, hi = offsets[i], offsets[i + 1]
            for h in range(s["q"]):
                k, v = (sequence(s[t], s["table"][i], first + hi - lo, h // group) for t in ("keys", "values"))
                for r in range(lo, hi, 2048):
                    end = min(hi, r + 2048)
                    logits = torch.mm(s["query"][r:end, h].double(), k.t()) / math.sqrt(s["d"])
                    hidden = torch.ones_like(logits, dtype=torch.bool).triu(first + r - lo + 1)
                    out[r:end, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ v
        return out

    return {"write": write, "decode": decode, "prompt": prompt}[case["op"]](prepare(case, seed))
