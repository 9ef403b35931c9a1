"""Operators of the cache held in 8 bits, each as a user calls it and in its plain form.

The cache (``leankv_b200.turboquant.byte_cache.ByteKVCache``) keeps keys and values in blocks of 16 tokens of one sequence and kv
head. A block has one scale, the smallest power of two 2^e (e >= -126) with ``|x| <= 127 * 2^e`` for all its numbers, and codes
``rint(x * 2^-e)``, half to even. A token that joins a block may raise e; the codes that are there are then rounded
once more. Operators, by ``kind``:

* ``update``: a prompt into an empty cache, and the cache's dense keys and values back (``ByteKVCache.update``);
* ``decode``: one query token per sequence over the cache (``decode_attention``);
* ``prompt``: causal attention of the last ``tokens`` tokens of every sequence (``prefill_attention``);
* ``sparse``: one query token per sequence over the ``blocks`` blocks that score best for it (``sparse_decode_attention``): the
  first ``sinks``, the last ``recent``, and those with the largest upper bound of the query heads' summed scores, taken from the
  blocks' largest and smallest codes a channel;
* ``steps``: tokens one by one, each appended and then answered from the cache (all of it, or ``blocks`` blocks), behind a
  prefix to which the cache is cut back first, and the dense cache at the end.

Sizes are those of the repository's benchmark configurations (8 kv heads, 4 query heads each, head size 128, contexts of 512 to
4096 tokens, 16 to 80 sequences) and of its mixer designs (head size 64, other groups), with odd lengths between and long
contexts beyond. Keys and values are N(0, 1) with four channels a head eight times as large, queries N(0, 1), as the benchmark's
generator makes them.
"""

from __future__ import annotations

import math

import torch

own = False                    # True: `run` calls the framework; False: the plain forms below
BLOCK = 16
SINKS, RECENT = 1, 2


# ── the cases ────────────────────────────────────────────────────────────────────────────────────────────────

def listed() -> list[dict]:
    base = dict(kv_heads=8, group=4, dim=128, dtype="float16")
    return [
        # the prompt of the headline decode loop goes into one layer's cache and is read back for a dense pass
        dict(base, name="update_512", kind="update", batch=1, tokens=512),
        # a batch of longer prompts, bf16, of a length that ends inside a block
        dict(base, name="update_16x2k", kind="update", batch=16, tokens=2011, dtype="bfloat16"),
        # the smallest call: one sequence that has just begun
        dict(base, name="decode_1x100", kind="decode", batch=1, tokens=101, more=0, longer=0),
        # one layer of a serving step: 16 sequences around 4096 tokens, not all of one length
        dict(base, name="decode_16x4k", kind="decode", batch=16, tokens=3851, more=490, longer=8),
        # long contexts, four sequences
        dict(base, name="decode_4x32k", kind="decode", batch=4, tokens=32781, more=0, longer=0, dtype="bfloat16"),
        # small heads in groups of seven, many sequences
        dict(name="decode_d64", kind="decode", batch=48, tokens=1500, more=333, longer=20, kv_heads=2, group=7, dim=64, dtype="bfloat16"),
        # the third chunk of 512 of a prompt and its like: everything before it is cached
        dict(base, name="prompt_512_at_3584", kind="prompt", batch=1, tokens=512, past=3584),
        # a whole prompt at once
        dict(base, name="prompt_4096", kind="prompt", batch=1, tokens=4096, past=0, dtype="bfloat16"),
        # a few sequences' short continuations (a question behind a document), odd everywhere
        dict(name="prompt_3x37", kind="prompt", batch=3, tokens=37, past=1003, kv_heads=4, group=3, dim=64, dtype="float16"),
        # a single very long sequence: 128 of its 8193 blocks are read
        dict(base, name="sparse_1x131k", kind="sparse", batch=1, tokens=131077, more=0, longer=0, blocks=128),
        # a batch around 8192 tokens of which 64 blocks are read
        dict(base, name="sparse_16x8k", kind="sparse", batch=16, tokens=7700, more=900, longer=7, blocks=64, dtype="bfloat16"),
        # a generation: 24 tokens for each of eight sequences
        dict(base, name="steps_8x1k", kind="steps", batch=8, tokens=1024, steps=24, blocks=0),
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number between the two, evenly over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["update", "decode", "decode", "prompt", "prompt", "sparse", "sparse", "steps"])
    dim = rng.choice([64, 128, 128])
    case = dict(kind=kind, kv_heads=rng.choice([1, 2, 3, 4, 8, 8]), group=rng.choice([1, 2, 3, 4, 4, 4, 5, 7, 8, 16]), dim=dim,
                dtype=rng.choice(["float16", "float16", "bfloat16", "bfloat16", "float32"]))
    if kind == "update":
        batch = _spread(rng, 1, 32)
        return dict(case, batch=batch, tokens=_spread(rng, 1, (16384 if case["dtype"] == "float32" else 32176) // batch))
    if kind == "decode":
        batch = _spread(rng, 1, 96)
        tokens = _spread(rng, 1, 98304 // batch)
        return dict(case, batch=batch, tokens=tokens, more=rng.randint(0, max(1, tokens // 4)), longer=rng.randint(0, batch))
    if kind == "prompt":
        batch, case["group"] = rng.choice([1, 1, 2, 5]), min(case["group"], 32 // case["kv_heads"])
        tokens = _spread(rng, 2, 2048 // batch)
        return dict(case, batch=batch, tokens=tokens, past=rng.choice([0, rng.randint(0, 100), _spread(rng, 1, 3000 // batch)]))
    if kind == "sparse":
        batch = _spread(rng, 1, 32)
        tokens = _spread(rng, 33, 98304 // batch)
        return dict(case, batch=batch, tokens=tokens, more=rng.randint(0, max(1, tokens // 4)), longer=rng.randint(0, batch),
                    blocks=_spread(rng, 4, 256))
    batch = _spread(rng, 1, 16)
    return dict(case, batch=batch, tokens=BLOCK * _spread(rng, 1, 512 // batch), steps=rng.randint(1, 24), blocks=rng.choice([0, 0, 8, 32]))


# ── inputs ───────────────────────────────────────────────────────────────────────────────────────────────────

def _lengths(case: dict) -> list[int]:
    """Tokens of each sequence that the cache holds when the timed call comes."""
    if case["kind"] == "prompt":
        return [case["past"] + case["tokens"]] * case["batch"]
    return [case["tokens"] + (case["more"] if b < case.get("longer", 0) else 0) for b in range(case["batch"])]


def _inputs(case: dict, seed: int) -> dict:
    """Keys, values and queries: ``k``, ``v`` [B, H, T, D] (T covers the longest sequence and the steps), ``q`` [B, G H, (tokens,) D]."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, h, d = getattr(torch, case["dtype"]), case["batch"], case["kv_heads"], case["dim"]
    t = max(_lengths(case)) + case.get("steps", 0)

    def vectors():
        x = torch.randn(b, h, t, d, generator=gen, device="cuda")
        large = torch.rand(h, d, generator=gen, device="cuda").topk(4, dim=1).indices
        return x.mul_(torch.ones(h, d, device="cuda").scatter_(1, large, 8.0)[:, None]).to(dtype)

    k, v = vectors(), vectors()
    n_q = {"prompt": case["tokens"], "steps": case.get("steps", 1)}.get(case["kind"], 1)
    q = torch.randn(b, h * case["group"], n_q, d, generator=gen, device="cuda").to(dtype)
    return {"k": k, "v": v, "q": q if case["kind"] in ("prompt", "steps") else q[:, :, 0].contiguous()}


def prepare(case: dict, seed: int) -> dict:
    x, n = _inputs(case, seed), _lengths(case)
    state = {"case": case, "q": x["q"]}
    held = 0 if case["kind"] == "update" else max(n)                 # tokens that are in the cache before the pass
    if held < x["k"].shape[2]:
        state["k"], state["v"] = (x[w][:, :, held:].contiguous() for w in "kv")
    if own:
        from leankv_b200.turboquant.byte_cache import ByteKVCache

        b, h = case["batch"], case["kv_heads"]
        pages = sum(-(-(t + case.get("steps", 0)) // BLOCK) for t in n) + 1
        cache = ByteKVCache(num_layers=1, num_kv_heads=h, num_q_heads=h * case["group"], head_dim=case["dim"], max_pages=pages,
                            dtype=x["k"].dtype, device="cuda")
        if held:
            cache.append(0, x["k"][:, :, :n[-1]], x["v"][:, :, :n[-1]])
            if max(n) > n[-1]:
                cache.append(0, x["k"][:case["longer"], :, n[-1]:held], x["v"][:case["longer"], :, n[-1]:held])
        return {**state, "cache": cache}
    state["lengths"] = torch.tensor(n, device="cuda")
    if held:
        # the second part of the longer sequences joins a block that is there already: rounded like that
        for w in "kv":
            codes, e = _quantize(x[w][:, :, :held].float(), state["lengths"])
            if max(n) > n[-1]:
                codes, e = _join(x[w][:, :, :held].float(), n[-1], state["lengths"], codes, e)
            state[w + "_codes"], state[w + "_scale"] = codes, _power(e)
        state["k_max"], state["k_min"] = _extremes(state["k_codes"], state["lengths"])
    return state


# ── one pass ─────────────────────────────────────────────────────────────────────────────────────────────────

def run(state: dict):
    case, q = state["case"], state["q"]
    kind = case["kind"]
    if own:
        cache = state["cache"]
        if kind == "update":
            cache.reset()
            return cache.update(state["k"], state["v"], 0)
        if kind == "decode":
            return cache.decode_attention(0, q)
        if kind == "prompt":
            return cache.prefill_attention(0, q)
        if kind == "sparse":
            return cache.sparse_decode_attention(0, q, blocks=case["blocks"], sinks=SINKS, recent=RECENT, return_blocks=True)
        cache.crop(case["tokens"])
        outs = []
        for i in range(case["steps"]):
            cache.append(0, state["k"][:, :, i:i + 1], state["v"][:, :, i:i + 1])
            if case["blocks"]:
                outs.append(cache.sparse_decode_attention(0, q[:, :, i], blocks=case["blocks"], sinks=SINKS, recent=RECENT))
            else:
                outs.append(cache.decode_attention(0, q[:, :, i]))
        return (torch.stack(outs, 2), *cache[0])
    lengths = state["lengths"]
    if kind == "update":
        return tuple(_dense(*_quantize(state[w].float(), lengths), state[w].shape[2]).to(q.dtype) for w in "kv")
    if kind == "steps":
        return _plain_steps(state)
    k, v = (_values(state[w + "_codes"], state[w + "_scale"]) for w in "kv")
    if kind == "decode":
        return _attend(q.float()[:, :, None], k, v, _visible(k, lengths)[:, None, None]).squeeze(2).to(q.dtype)
    if kind == "prompt":
        at = torch.arange(case["past"], case["past"] + case["tokens"], device=q.device)
        return _attend(q.float(), k, v, (torch.arange(k.shape[2] * BLOCK, device=q.device) <= at[:, None])[None, None]).to(q.dtype)
    out, chosen = _plain_sparse(q.float(), k, v, state["k_max"], state["k_min"], state["k_scale"], lengths, case["blocks"])
    return out.to(q.dtype), chosen


# ── plain forms: elementary operations in 32 bits ────────────────────────────────────────────────────────────

def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e of whole exponents from -126 to 127, put together from its bits: a power function may be a rounding off."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _exponent(amax: torch.Tensor, most: int) -> torch.Tensor:
    """The smallest e >= -126 with ``amax <= most * 2^e``; ``most`` is a power of two less one."""
    mant, e = torch.frexp(amax)
    bits = most.bit_length()
    e = e - bits + (mant > most / 2 ** bits)
    return torch.where(amax > 0, e, -126).clamp(min=-126).to(torch.int32)


def _real(codes: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
    """Which slots of blocks [B, H, N, 16, D] hold a token, [B, 1, N, 16, 1]."""
    at = torch.arange(codes.shape[2] * BLOCK, device=codes.device).view(1, 1, -1, BLOCK, 1)
    return at < lengths.view(-1, 1, 1, 1, 1)


def _quantize(x: torch.Tensor, lengths: torch.Tensor):
    """Vectors [B, H, T, D] that come at once as codes [B, H, N, 16, D] and exponents [B, H, N]."""
    n = -(-x.shape[2] // BLOCK)
    x = torch.nn.functional.pad(x, (0, 0, 0, n * BLOCK - x.shape[2])).view(*x.shape[:2], n, BLOCK, x.shape[3])
    x = x * _real(x, lengths)
    e = _exponent(x.abs().amax(dim=(3, 4)), 127)
    return torch.round(x * _power(-e)[..., None, None]).to(torch.int8), e


def _join(x: torch.Tensor, first: int, lengths: torch.Tensor, codes: torch.Tensor, e: torch.Tensor):
    """Codes and exponents when the tokens from ``first`` on came in a second call: the block that ``first`` falls into was
    rounded with its first tokens' scale before."""
    if first % BLOCK == 0:
        return codes, e
    j = first // BLOCK
    early, e0 = _quantize(x[:, :, j * BLOCK:first], torch.full_like(lengths, first - j * BLOCK))
    grown = torch.maximum(e[:, :, j], e0[:, :, 0])
    late = x[:, :, j * BLOCK:(j + 1) * BLOCK] * (torch.arange(j * BLOCK, min((j + 1) * BLOCK, x.shape[2]), device=x.device)[:, None] >= first)
    late = late * (lengths > first).view(-1, 1, 1, 1)
    both = torch.round(early[:, :, 0].float() * _power(e0[:, :, 0] - grown)[..., None, None])
    both[:, :, :late.shape[2]] += torch.round(late * _power(-grown)[..., None, None])
    codes, e = codes.clone(), e.clone()
    codes[:, :, j], e[:, :, j] = both.to(torch.int8), grown
    return codes, e


def _values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return codes.float() * scale[..., None, None]


def _dense(codes: torch.Tensor, e: torch.Tensor, tokens: int) -> torch.Tensor:
    return _values(codes, _power(e)).flatten(2, 3)[:, :, :tokens]


def _extremes(codes: torch.Tensor, lengths: torch.Tensor):
    """The largest and the smallest code of each channel among a block's tokens, [B, H, N, D]."""
    real = _real(codes, lengths)
    c = codes.short()
    return c.where(real, -128).amax(3).to(torch.int8), c.where(real, 127).amin(3).to(torch.int8)


def _visible(k: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
    return torch.arange(k.shape[2] * BLOCK, device=k.device) < lengths[:, None]


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, see: torch.Tensor) -> torch.Tensor:
    """q [B, G H, Q, D] over blocks k, v [B, H, N, 16, D] where ``see`` (broadcast over [B, H, Q, tokens]) allows; [B, G H, Q, D]."""
    b, h, d = k.shape[0], k.shape[1], k.shape[-1]
    q = q.view(b, h, -1, q.shape[2], d)
    s = (q.flatten(2, 3) @ k.flatten(2, 3).transpose(2, 3)).view(*q.shape[:4], -1) / math.sqrt(d)
    s = s.masked_fill(~see.unsqueeze(2), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return (p.flatten(2, 3) @ v.flatten(2, 3)).view(b, -1, q.shape[3], d)


def _choose(q: torch.Tensor, k_max, k_min, k_scale, lengths, blocks: int) -> torch.Tensor:
    """The blocks that each sequence and kv head reads, ascending, then -1: int32 [B, H, blocks]. Sums of whole numbers below
    2^31 times a power of two: formed in 64 bits, rounded to 32 once, so that ties are ties everywhere."""
    b, h, n = k_scale.shape
    qg = q.view(b, h, -1, q.shape[-1])
    f = _exponent(qg.abs().amax(dim=(2, 3)), 2047)
    i = torch.round(qg * _power(-f)[..., None, None]).double()
    up, down = i.clamp(min=0).sum(2), i.clamp(max=0).sum(2)
    u = (up[:, :, None] * k_max.double() + down[:, :, None] * k_min.double()).sum(-1)
    score = u.float() * k_scale
    at, have = torch.arange(n, device=q.device), (lengths + BLOCK - 1) // BLOCK
    have = have.view(-1, 1, 1)
    score = score.masked_fill((at < SINKS) | (at >= have - RECENT), math.inf).masked_fill(at >= have, -math.inf)
    score = torch.nn.functional.pad(score, (0, max(0, blocks - n)), value=-math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :blocks]
    best = best.masked_fill(best >= have, n + blocks).sort(-1).values
    return best.masked_fill(best >= n, -1).to(torch.int32)


def _plain_sparse(q, k, v, k_max, k_min, k_scale, lengths, blocks: int):
    chosen = _choose(q, k_max, k_min, k_scale, lengths, blocks)
    at = chosen.long().clamp(min=0)[..., None, None]
    k, v = (x.gather(2, at.expand(-1, -1, -1, BLOCK, x.shape[-1])) for x in (k, v))
    pos = at[..., 0] * BLOCK + torch.arange(BLOCK, device=q.device)
    see = ((pos < lengths.view(-1, 1, 1, 1)) & (chosen[..., None] >= 0)).flatten(2).unsqueeze(2)
    return _attend(q[:, :, None], k, v, see).squeeze(2), chosen


def _plain_steps(state: dict):
    case, q = state["case"], state["q"]
    b, h, d, blocks = case["batch"], case["kv_heads"], case["dim"], case["blocks"]
    n0, extra = case["tokens"] // BLOCK, -(-case["steps"] // BLOCK)
    codes, e = {}, {}
    for w in "kv":
        more = torch.zeros(b, h, extra, BLOCK, d, dtype=torch.int8, device=q.device)
        codes[w] = torch.cat([state[w + "_codes"], more], 2)
        e[w] = torch.cat([torch.frexp(state[w + "_scale"])[1] - 1, torch.full((b, h, extra), -126, device=q.device, dtype=torch.int32)], 2)
    outs = []
    for i in range(case["steps"]):                     # a token sees what the ones before it have left
        j, slot = n0 + i // BLOCK, i % BLOCK
        for w in "kv":
            x = state[w][:, :, i].float()
            old = e[w][:, :, j].clone()
            new = torch.maximum(old, _exponent(x.abs().amax(-1), 127))
            kept = torch.round(codes[w][:, :, j].float() * _power((old - new).clamp(min=-126))[..., None, None])
            kept[:, :, slot] = torch.round(x * _power(-new)[..., None])
            codes[w][:, :, j], e[w][:, :, j] = kept.to(torch.int8), new
        lengths = state["lengths"] + i + 1
        k, v = (_values(codes[w], _power(e[w])) for w in "kv")
        if blocks:
            out, _ = _plain_sparse(q[:, :, i].float(), k, v, *_extremes(codes["k"], lengths), _power(e["k"]), lengths, blocks)
        else:
            out = _attend(q[:, :, i:i + 1].float(), k, v, _visible(k, lengths)[:, None, None]).squeeze(2)
        outs.append(out)
    n = case["tokens"] + case["steps"]
    return (torch.stack(outs, 2).to(q.dtype), *(_dense(codes[w], e[w], n).to(q.dtype) for w in "kv"))


# ── what a pass cannot do without ────────────────────────────────────────────────────────────────────────────

def work(case: dict) -> dict:
    size = {"float16": 2, "bfloat16": 2, "float32": 4}[case["dtype"]]
    h, g, d, b, kind = case["kv_heads"], case["group"], case["dim"], case["batch"], case["kind"]
    n = _lengths(case)
    block = 2 * BLOCK * d + 8                          # codes and scales of a block, keys and values
    vectors = lambda tokens: 2 * tokens * h * d * size # keys and values as numbers
    count = lambda lengths: sum(-(-t // BLOCK) for t in lengths)
    if kind == "update":
        return {"bytes": 2 * vectors(sum(n)) + count(n) * h * (block + 2 * d), "flops": 2.0 * 2 * sum(n) * h * d}
    if kind == "decode":
        return {"bytes": count(n) * h * block + 2 * b * h * g * d * size, "flops": 4.0 * sum(n) * h * g * d}
    if kind == "prompt":
        t, past = case["tokens"], case["past"]
        seen = b * (t * past + t * (t + 1) // 2)
        return {"bytes": count(n) * h * block + 2 * b * t * h * g * d * size, "flops": 4.0 * seen * h * g * d}

    def sparse(lengths):
        read = sum(min(case["blocks"], -(-t // BLOCK)) for t in lengths)
        return {"bytes": h * (count(lengths) * (2 * d + 4) + read * block) + 2 * b * h * g * d * size,
                "flops": h * d * (4.0 * count(lengths) + 4.0 * BLOCK * read * g)}

    if kind == "sparse":
        return sparse(n)
    total = {"bytes": vectors(b * (case["tokens"] + case["steps"])) + vectors(b * case["steps"]), "flops": 0.0}
    for i in range(case["steps"]):
        now = [t + i + 1 for t in n]
        one = sparse(now) if case["blocks"] else {"bytes": count(now) * h * block + 2 * b * h * g * d * size,
                                                  "flops": 4.0 * sum(now) * h * g * d}
        total = {m: total[m] + one[m] for m in total}
    return total


# ── the definitions in 64 bits ───────────────────────────────────────────────────────────────────────────────

def _two(e: torch.Tensor) -> torch.Tensor:
    """2^e, e whole, in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


class _Exact:
    """The cache of one case as its definition has it, written call by call."""

    def __init__(self, case: dict, slots: int):
        n = -(-slots // BLOCK)
        shape = (case["batch"], case["kv_heads"], n)
        self.code = {w: torch.zeros(*shape, BLOCK, case["dim"], dtype=torch.float64, device="cuda") for w in "kv"}
        self.exp = {w: torch.full(shape, -126.0, dtype=torch.float64, device="cuda") for w in "kv"}
        self.n = [0] * case["batch"]

    @staticmethod
    def least(amax: torch.Tensor, most: float) -> torch.Tensor:
        """The smallest whole e >= -126 with amax <= most 2^e."""
        e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / most)).clamp(min=-126)
        e = torch.where(amax <= most * _two(e - 1), e - 1, e)               # the logarithm may have rounded either way
        return torch.where(amax > most * _two(e), e + 1, e).clamp(min=-126)

    def append(self, k: torch.Tensor, v: torch.Tensor):
        """Tokens [B', H, T, D] for the first B' sequences, which are of one length."""
        seqs, t, first = k.shape[0], k.shape[2], self.n[0]
        for w, x in (("k", k.double()), ("v", v.double())):
            for j in range(first // BLOCK, -(-(first + t) // BLOCK)):
                lo, hi = max(first, j * BLOCK), min(first + t, (j + 1) * BLOCK)
                new = x[:, :, lo - first:hi - first]
                old = self.exp[w][:seqs, :, j] if first > j * BLOCK else torch.full_like(self.exp[w][:seqs, :, j], -126.0)
                e = torch.maximum(old, self.least(new.abs().amax(dim=(2, 3)), 127.0))
                block = self.code[w][:seqs, :, j]
                block.copy_(torch.round(block * _two(old - e)[..., None, None]))
                block[:, :, lo - j * BLOCK:hi - j * BLOCK] = torch.round(new / _two(e)[..., None, None])
                self.exp[w][:seqs, :, j] = e
        for s in range(seqs):
            self.n[s] += t

    def numbers(self, w: str, s: int) -> torch.Tensor:
        """Keys or values of a sequence, [H, tokens, D]."""
        return (self.code[w][s] * _two(self.exp[w][s])[..., None, None]).flatten(1, 2)[:, :self.n[s]]

    def dense(self, w: str) -> torch.Tensor:
        return torch.stack([self.numbers(w, s) for s in range(len(self.n))])

    def attend(self, s: int, q: torch.Tensor, at: int, chosen=None) -> torch.Tensor:
        """Queries [H, G, Q, D] of a sequence, the first one at position ``at``; ``chosen`` [H, K]: the blocks that may be seen."""
        k, v = self.numbers("k", s), self.numbers("v", s)
        pos = torch.arange(k.shape[1], device=k.device)
        see = (pos <= at + torch.arange(q.shape[2], device=k.device)[:, None]).expand(k.shape[0], -1, -1)
        if chosen is not None:
            see = see & ((pos // BLOCK)[None, :, None] == chosen[:, None, :].long()).any(-1)[:, None]
        out = torch.empty_like(q)
        for head in range(q.shape[0]):
            w = torch.einsum("gqd,td->gqt", q[head], k[head]) * q.shape[-1] ** -0.5
            w = torch.softmax(w.where(see[head], -math.inf), -1)
            out[head] = torch.einsum("gqt,td->gqd", w, v[head])
        return out

    def choose(self, s: int, q: torch.Tensor, blocks: int) -> torch.Tensor:
        """The blocks that queries [H, G, D] read, [H, blocks]."""
        n = -(-self.n[s] // BLOCK)
        out = torch.full((q.shape[0], blocks), -1, dtype=torch.int32, device=q.device)
        if n <= blocks:
            out[:, :n] = torch.arange(n, dtype=torch.int32, device=q.device)
            return out
        whole = torch.round(q / _two(self.least(q.abs().amax(dim=(1, 2)), 2047.0))[:, None, None])
        code, tail = self.code["k"][s, :, :n], self.n[s] - (n - 1) * BLOCK
        big, small = code.amax(2), code.amin(2)
        big[:, -1], small[:, -1] = code[:, -1, :tail].amax(1), code[:, -1, :tail].amin(1)
        bound = torch.maximum(whole[:, :, None] * big[:, None], whole[:, :, None] * small[:, None]).sum(dim=(1, 3))
        score = (bound.float() * _two(self.exp["k"][s, :, :n]).float()).cpu().tolist()
        for head, row in enumerate(score):
            free = sorted(range(SINKS, n - RECENT), key=lambda j: (-row[j], j))[:blocks - SINKS - RECENT]
            picked = sorted([*range(SINKS), *free, *range(n - RECENT, n)])
            out[head] = torch.tensor(picked, dtype=torch.int32)
        return out


def exact(case: dict, seed: int):
    x, n, kind = _inputs(case, seed), _lengths(case), case["kind"]
    b, h, g, d = case["batch"], case["kv_heads"], case["group"], case["dim"]
    cache = _Exact(case, x["k"].shape[2])
    cache.append(x["k"][:, :, :n[-1]], x["v"][:, :, :n[-1]])
    if max(n) > n[-1]:
        cache.append(x["k"][:case["longer"], :, n[-1]:max(n)], x["v"][:case["longer"], :, n[-1]:max(n)])
    if kind == "update":
        return cache.dense("k"), cache.dense("v")
    q = x["q"].double().view(b, h, g, -1, d)

    def answer(at, i, blocks):
        outs, picked = [], []
        for s in range(b):
            one = q[s] if i is None else q[s, :, :, i:i + 1]
            chosen = cache.choose(s, one[:, :, 0], blocks) if blocks else None
            outs.append(cache.attend(s, one, at(s), chosen).flatten(0, 1))
            picked.append(chosen)
        return torch.stack(outs), picked

    if kind == "decode":
        return answer(lambda s: n[s] - 1, None, 0)[0].squeeze(2)
    if kind == "prompt":
        return answer(lambda s: case["past"], None, 0)[0]
    if kind == "sparse":
        out, picked = answer(lambda s: n[s] - 1, None, case["blocks"])
        return out.squeeze(2), torch.stack(picked)
    outs = []
    for i in range(case["steps"]):
        cache.append(x["k"][:, :, n[0] + i:n[0] + i + 1], x["v"][:, :, n[0] + i:n[0] + i + 1])
        outs.append(answer(lambda s: n[s] + i, i, case["blocks"])[0])
    return torch.cat(outs, 2), cache.dense("k"), cache.dense("v")
