"""The 8-bit paged cache on the GPU against its definition in 64 bits (``oracle/bytes.py``).

Codes, scales, bounds and chosen blocks have to be equal: every rounding in them is of an exact number. Attention: the kernels
form scores, weights and sums in 32 bits from exact codes and a query of 22 bits or more, weights enter as two 11-bit parts. A score is a sum of
``dim`` products in fp32 (tensor-core sums drop bits of 2^-22 of the largest term at worst), |s| up to some 20 in these tests, so a weight is off by at most
2^-22 * 20 * 2 ~ 1e-5 of itself, and so is an output relative to its row; then one rounding to the output type, eps / 2 at most. Bound: relative 2-norm
over a row ``eps / 2 + 2e-5``.

The prompt kernel rounds each weight to fp16 (relative 2^-11 at most, both ways alike) before the value product. Its part of a row's error is at most
2^-11 sum_t w_t |v_t|, which the rows of these tests, whose values have random signs, are not far above: ``|out| >= |v| / sqrt(n)`` in the mean and the errors
add up like the values do, so that relative to the row it stays below 2^-11 again with a factor of 2 for small rows: bound ``eps / 2 + 2e-5 + 2^-10``.
"""

import math

import pytest
import torch

from leankv_b200 import _native
from leankv_b200.turboquant.byte_cache import ByteKVCache
from oracle import bytes as obytes

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def vectors(gen, batch, heads, tokens, dim, dtype, large=True):
    x = torch.randn(batch, heads, tokens, dim, generator=gen)
    if large:
        x[..., ::dim // 4] *= 8
    return x.to(dtype)


def row_errors(got, want):
    """Relative 2-norm of each row's error; rows that should be zero have to be."""
    got, want = got.double().cpu().flatten(0, -2), want.flatten(0, -2)
    size = want.norm(dim=-1)
    assert bool((got[size == 0] == 0).all())
    return ((got - want).norm(dim=-1) / size.clamp_min(1e-300))[size > 0]


def close(got, want, dtype, weights=False):
    err = row_errors(got, want)
    assert got.dtype == dtype
    bound = torch.finfo(dtype).eps / 2 + 2e-5 + (2.0 ** -10 if weights else 0.0)
    assert len(err) == 0 or float(err.max()) <= bound, (float(err.max()), bound)


class Pair:
    """A cache on the GPU and its definition, given the same tokens."""

    def __init__(self, batch, heads, group, dim, dtype, pages=64, layers=1, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.batch, self.heads, self.group, self.dim, self.dtype = batch, heads, group, dim, dtype
        self.cache = ByteKVCache(num_layers=layers, num_kv_heads=heads, num_q_heads=heads * group, head_dim=dim, max_pages=pages, dtype=dtype, device=DEV)
        self.plain = obytes.Cache(batch, heads, dim)

    def append(self, tokens, batch=None, scale=1.0, layer=0):
        k, v = ((vectors(self.gen, batch or self.batch, self.heads, tokens, self.dim, torch.float32) * scale).to(self.dtype) for _ in range(2))
        self.cache.append(layer, k.to(DEV), v.to(DEV))
        self.plain.append(k, v)

    def queries(self, tokens=None):
        shape = (self.batch, self.heads * self.group) + (() if tokens is None else (tokens,)) + (self.dim,)
        return torch.randn(shape, generator=self.gen).to(self.dtype)

    def check_pages(self, layer=0):
        for b in range(self.batch):
            if self.plain.n[b] == 0:
                continue
            for which in range(2):
                codes, scales = self.cache.unpack_sequence(layer, b, which)
                assert torch.equal(codes.cpu().double(), self.plain.codes(b, which))
                assert torch.equal(scales.cpu().double().nan_to_num(-1.0), self.plain.scales(b, which).nan_to_num(-1.0))
            ids = self.cache._block_table[b, :-(-self.plain.n[b] // 16)].long()
            rec = self.cache.bounds[layer][ids].cpu()
            for h in range(self.heads):
                for j, block in enumerate(self.plain.blocks[0][b][h]):
                    got = rec[j, h, :2 * self.dim].contiguous().view(torch.int8).double()
                    assert torch.equal(got[:self.dim], block.codes.amax(0)) and torch.equal(got[self.dim:], block.codes.amin(0))

    def check_decode(self):
        q = self.queries()
        got = self.cache.decode_attention(0, q.to(DEV))
        want = torch.stack([self.plain.attend(b, q[b, :, None])[:, 0] for b in range(self.batch)])
        close(got, want, self.dtype)
        assert self.cache.kernel_status() == 0

    def check_prompt(self, tokens):
        """Both kernels, whichever the work would choose."""
        q = self.queries(tokens)
        want = torch.stack([self.plain.attend(b, q[b]) for b in range(self.batch)])
        for work in (0, 1 << 60):
            self.cache._prompt_work = work
            got = self.cache.prefill_attention(0, q.to(DEV))
            close(got, want, self.dtype, weights=work == 0 and self.dtype != F32)
            assert self.cache.kernel_status() == 0

    def check_sparse(self, blocks, sinks=1, recent=2):
        q = self.queries()
        got, chosen = self.cache.sparse_decode_attention(0, q.to(DEV), blocks, sinks, recent, return_blocks=True)
        for b in range(self.batch):
            want = self.plain.choose(b, q[b], blocks, sinks, recent)
            assert torch.equal(chosen[b].cpu(), want), (b, chosen[b].cpu(), want)
            close(got[b], self.plain.attend(b, q[b, :, None], want)[:, 0], self.dtype)
        again = self.cache.sparse_decode_attention(0, q.to(DEV), blocks, sinks, recent)
        assert torch.equal(again, got) and self.cache.kernel_status() == 0
        return chosen


# ── pages ────────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("chunks", [(1,), (16,), (17, 1, 1, 13), (5, 40, 3), (1, 2, 1, 33, 1, 1)])
def test_codes_scales_and_bounds_are_those_of_the_definition(dtype, dim, chunks):
    p = Pair(3, 2, 2, dim, dtype, seed=sum(chunks) + dim)
    for i, n in enumerate(chunks):
        p.append(n, scale=[1.0, 3.0, 1e-3, 40.0][i % 4])
        p.check_pages()
    keys, values = p.cache[0]
    for b in range(3):
        for got, which in ((keys, 0), (values, 1)):
            assert got.dtype == dtype and torch.equal(got[b].cpu(), p.plain.values(b, which).to(dtype))


def test_ragged_sequences_keep_their_own_scales():
    p = Pair(4, 3, 1, 64, BF16)
    p.append(21)
    p.append(9, batch=2, scale=7.0)
    p.append(1, batch=3, scale=0.1)
    p.append(2, scale=30.0)
    p.check_pages()
    keys, _ = p.cache[0]
    assert keys.shape == (4, 3, 33, 64)
    assert bool((keys[3, :, 23:] == 0).all()) and bool((keys[2, :, 24:] == 0).all())
    p.check_decode()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_smallest_and_largest_magnitudes(dtype):
    p = Pair(1, 2, 1, 64, dtype)
    for scale in (0.0, 1e-40, 1e-30, 1e30):
        p.append(16, scale=scale)
    p.append(3, scale=0.0)
    p.append(2, scale=1e-20)
    p.check_pages()


def test_an_fp16_block_whose_largest_code_stands_for_more_than_fp16_holds():
    p = Pair(1, 1, 1, 64, F16)
    k = torch.full((1, 1, 4, 64), 65504.0, dtype=F16)
    p.cache.append(0, k.to(DEV), (-k).to(DEV))
    p.plain.append(k, -k)
    p.check_pages()
    keys, values = p.cache[0]
    assert bool((keys == 65504).all()) and bool((values == -65504).all())


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", [0, 1])
def test_a_block_that_holds_no_number_answers_nobody_who_sees_it(bad, which):
    p = Pair(2, 2, 2, 64, BF16)
    p.append(32)
    k, v = (vectors(p.gen, 2, 2, 20, 64, BF16) for _ in range(2))
    (k, v)[which][0, 1, 2, 5] = bad                    # position 34 of sequence 0, head 1: block 2
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    p.check_pages()
    q = p.queries()
    got = p.cache.decode_attention(0, q.to(DEV)).cpu()
    assert bool(got[0, 2:].isnan().all())
    q20 = p.queries(20)
    q40 = p.queries(40)                                # positions 12 .. 51; those before 32 do not see block 2
    cut = obytes.Cache(2, 2, 64)
    cut.blocks = [[[row[:2] for row in seq] for seq in side] for side in p.plain.blocks]
    cut.n = [32, 32]
    for work in (0, 1 << 60):                          # either kernel
        p.cache._prompt_work = work
        prompt = p.cache.prefill_attention(0, q20.to(DEV)).cpu()
        assert bool(prompt[0, 2:].isnan().all())       # every token of the chunk shares the block or comes behind it
        wide = p.cache.prefill_attention(0, q40.to(DEV))
        assert bool(wide[0, 2:, 20:].isnan().all())
        want = [p.plain.attend(b, q40[b]) for b in range(2)]
        close(wide[0, :2], want[0][:2], BF16, work == 0)
        close(wide[1], want[1], BF16, work == 0)
        close(wide[0, 2:, :20], cut.attend(0, q40[0, :, :20])[2:], BF16, work == 0)
    # the block counts as the best one of all
    sparse, chosen = p.cache.sparse_decode_attention(0, q.to(DEV), 3, 0, 1, return_blocks=True)
    if which == 0:
        assert 2 in chosen[0, 1].tolist() and bool(sparse[0, 2:].isnan().all())
    p.append(30)                                       # the block is full by now and stays as it is
    p.check_pages()
    assert p.cache.kernel_status() == 0


def test_crop_gives_pages_back_and_the_next_tokens_join_what_is_left():
    p = Pair(3, 2, 1, 128, F16, pages=24)
    p.append(50)
    p.append(20, batch=1)
    used = p.cache.get_pages_used()
    for keep, then in ((64, 3), (41, 9), (32, 1), (17, 2), (0, 33)):
        p.cache.crop(keep)
        p.plain.crop(keep)
        assert p.cache._seq_lengths == p.plain.n
        assert p.cache.get_pages_used() == sum(-(-n // 16) for n in p.plain.n) <= used
        if keep:
            p.check_decode()
        p.append(then, scale=2.0)
        p.check_pages()
        p.check_decode()
    p.cache.crop(-3)
    assert p.cache.get_seq_length() == max(p.plain.n) - 3 and p.cache.page_table_status() == 0
    free = p.cache._free_stack[:p.cache._free_count].tolist()
    held = [i for b, n in enumerate(p.cache._seq_lengths) for i in p.cache._block_table[b, :-(-n // 16)].tolist()]
    assert sorted(free + held) == list(range(24)) and int(p.cache._free_top) == len(free)


def test_crop_takes_back_what_was_seen():
    p = Pair(2, 1, 1, 64, F16)
    p.append(50)
    for keep, seen in ((60, 50), (41, 41), (-3, 38), (0, 0)):
        p.cache.crop(keep)
        assert p.cache.seen_tokens == p.cache.get_seq_length() == seen
    p.append(7, batch=1)
    assert p.cache.seen_tokens == p.cache.get_seq_length() == 7


def test_a_full_pool_is_refused_and_leaves_the_cache_as_it_was():
    p = Pair(2, 1, 1, 64, F16, pages=6)
    p.append(40)
    with pytest.raises(RuntimeError, match="out of pages"):
        p.append(20)
    assert p.cache._seq_lengths == [40, 40] and p.cache.get_pages_used() == 6
    p.plain.n = [40, 40]
    p.check_pages()
    p.check_decode()
    p.cache.reset()
    assert p.cache.get_pages_used() == 0 and p.cache.get_seq_length() == 0
    p.plain = obytes.Cache(2, 1, 64)
    p.append(48)
    p.check_pages()


def test_arguments_that_do_not_fit_are_refused():
    p = Pair(2, 2, 3, 64, F16, layers=2)
    k = torch.zeros(2, 2, 4, 64, dtype=F16, device=DEV)
    for bad in (k[:, :1], k[..., :32], k[0], torch.zeros(1025, 2, 1, 64, dtype=F16, device=DEV), k[:0]):
        with pytest.raises(RuntimeError):
            p.cache.append(0, bad, bad)
    with pytest.raises(RuntimeError):
        p.cache.append(0, k, k[:, :, :3])
    with pytest.raises(RuntimeError, match="layers"):
        p.cache.append(2, k, k)
    with pytest.raises(RuntimeError, match="layer 0"):
        p.cache.append(1, k, k)
    assert p.cache._seq_lengths in ([], [0, 0])
    p.cache.append(0, k, k)
    with pytest.raises(RuntimeError, match="appended"):
        p.cache.prefill_attention(0, torch.zeros(2, 6, 5, 64, dtype=F16, device=DEV))
    for bad in (torch.zeros(2, 5, 64, dtype=F16, device=DEV), torch.zeros(2, 6, 32, dtype=F16, device=DEV), torch.zeros(6, 64, dtype=F16, device=DEV)):
        with pytest.raises(RuntimeError):
            p.cache.decode_attention(0, bad)


# ── attention ────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("group", [1, 4, 7, 8, 9, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_attention_for_every_group_and_type(dtype, group, dim):
    p = Pair(3, 2, group, dim, dtype, seed=group)
    p.append(37)
    p.append(70, batch=2)
    p.append(1, batch=1)
    p.check_decode()


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 64, 127, 129, 500, 1025])
def test_decode_attention_for_lengths_around_blocks_and_shares(tokens):
    p = Pair(2, 1, 4, 128, F16, pages=200, seed=tokens)
    p.append(tokens)
    p.check_decode()


def test_sequences_without_tokens_get_zeros():
    p = Pair(5, 2, 3, 64, BF16)
    p.append(20, batch=2)
    p.check_decode()                                   # sequences 2 .. 4 are empty
    p.cache.crop(0)
    p.plain.crop(0)
    p.check_decode()


@pytest.mark.parametrize("batch, heads, tokens", [(1, 1, 9000), (1, 8, 3000), (7, 3, 1111), (70, 2, 90)])
def test_shares_of_many_thread_blocks_add_up(batch, heads, tokens):
    p = Pair(batch, heads, 4, 128, F16, pages=batch * (tokens // 16 + 6) + 8, seed=batch)
    p.append(tokens)
    p.append(73, batch=(batch + 1) // 2)
    p.check_decode()
    q = p.queries().to(DEV)
    first = p.cache.decode_attention(0, q)
    assert all(torch.equal(p.cache.decode_attention(0, q), first) for _ in range(5))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim, group, heads", [(64, 3, 2), (128, 4, 1), (128, 7, 2), (64, 16, 1)])
@pytest.mark.parametrize("past, tokens", [(0, 2), (0, 33), (5, 12), (70, 31), (250, 5)])
def test_prompt_attention_is_causal(dtype, dim, group, heads, past, tokens):
    p = Pair(2, heads, group, dim, dtype, seed=past + tokens)
    if past:
        p.append(past)
    p.append(tokens)
    p.check_prompt(tokens)


@pytest.mark.parametrize("dtype, dim, group, heads, past, tokens", [
    (F16, 128, 4, 2, 0, 260), (BF16, 128, 4, 1, 700, 130), (F16, 64, 3, 3, 129, 200), (BF16, 64, 16, 1, 1000, 40), (F16, 128, 1, 2, 2100, 300),
    (BF16, 128, 7, 1, 383, 129), (F16, 64, 5, 1, 4000, 64)])
def test_prompt_attention_over_several_tiles_and_shares(dtype, dim, group, heads, past, tokens):
    p = Pair(2, heads, group, dim, dtype, pages=600, seed=past + tokens)
    if past:
        p.append(past)
    p.append(50, batch=1)
    p.append(tokens)
    p.check_prompt(tokens)
    q = p.queries(tokens).to(DEV)
    p.cache._prompt_work = 0
    first = p.cache.prefill_attention(0, q)
    assert all(torch.equal(p.cache.prefill_attention(0, q), first) for _ in range(3))


@pytest.mark.parametrize("dtype, dim, group, heads, past, tokens", [
    (F16, 128, 4, 1, 8200, 20), (BF16, 64, 7, 2, 16390, 40), (F16, 128, 16, 2, 9000, 9), (BF16, 128, 3, 1, 12345, 1)])
def test_prompt_attention_of_few_rows_behind_many_pages(dtype, dim, group, heads, past, tokens):
    """Keys shared by several clusters, whose sums meet in the workspace: twice, the second time on what the first has left there."""
    p = Pair(1, heads, group, dim, dtype, pages=(past + tokens) // 16 + 1, seed=past)
    p.append(past)
    p.append(tokens)
    q = p.queries(tokens)
    want = p.plain.attend(0, q[0])[None]
    p.cache._prompt_work = 0
    first = p.cache.prefill_attention(0, q.to(DEV))
    again = p.cache.prefill_attention(0, q.to(DEV))
    close(first, want, dtype, weights=True)
    assert torch.equal(first, again) and p.cache.kernel_status() == 0


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0])
def test_prompt_attention_on_values_of_different_magnitudes(scale):
    """Value blocks whose scales differ by up to 2^20 under the largest one, which the weights do not prefer."""
    p = Pair(1, 1, 2, 64, BF16, pages=80)
    for i in range(20):
        k = vectors(p.gen, 1, 1, 16, 64, BF16, large=False)
        v = (vectors(p.gen, 1, 1, 16, 64, torch.float32, large=False) * scale * 2.0 ** -(i % 5 * 5)).to(BF16)
        p.cache.append(0, k.to(DEV), v.to(DEV))
        p.plain.append(k, v)
    p.check_prompt(200)


@pytest.mark.parametrize("kind, dtype, dim, group, heads, past, tokens", [
    ("later", BF16, 128, 4, 1, 0, 300), ("later", F16, 64, 4, 2, 0, 200), ("later", BF16, 64, 3, 1, 37, 700), ("mixed", BF16, 64, 2, 1, 90, 150),
    ("mixed", BF16, 128, 4, 1, 0, 600), ("mixed", BF16, 128, 16, 1, 2000, 40), ("mixed", BF16, 128, 4, 1, 8200, 20), ("outweighed", BF16, 64, 7, 1, 500, 130),
    ("outweighed", BF16, 128, 4, 1, 0, 700), ("zeros", BF16, 128, 4, 1, 0, 500), ("zeros", F16, 64, 2, 1, 3000, 30), ("far", BF16, 128, 2, 1, 0, 400),
    ("far", BF16, 64, 2, 1, 1100, 30), ("far, near", BF16, 128, 2, 1, 0, 400), ("far, near", BF16, 64, 2, 1, 1100, 30), ("cliff", BF16, 64, 4, 1, 0, 400),
    ("cliff", BF16, 128, 2, 1, 1000, 50), ("own block", BF16, 64, 2, 1, 0, 270), ("own block", BF16, 128, 4, 1, 600, 30), ("own block", BF16, 64, 2, 1, 1390, 30),
    ("rare", BF16, 128, 4, 1, 0, 500), ("rare", BF16, 64, 3, 1, 1700, 40), ("first", BF16, 128, 2, 1, 0, 420), ("first", BF16, 64, 4, 1, 1500, 30),
    ("creeping", BF16, 128, 2, 1, 0, 800), ("creeping", BF16, 64, 2, 1, 2000, 20), ("silent", BF16, 128, 2, 1, 0, 500), ("silent", BF16, 64, 2, 1, 1500, 30)])
def test_a_prompt_row_goes_by_the_values_that_it_sees(kind, dtype, dim, group, heads, past, tokens):
    """Values of any spread: a row of small ones ahead of a later token's large ones; large ones whose weights leave the small ones what counts; blocks
    of zeros that take weight. A term is 2^-11 off for its weight's rounding, whatever its value, or 2^-24 of what the row's largest weight could bring in its block's
    scale: the bound that ``close`` has."""
    n = past + tokens
    p = Pair(1, heads, group, dim, dtype, pages=n // 16 + 2, seed=n + dim)
    k, v = (vectors(p.gen, 1, heads, n, dim, F32, large=False) for _ in range(2))
    q = p.queries(tokens)
    block = torch.arange(n) // 16
    if kind == "later":
        small, large = (2.0 ** -10, 2.0 ** 13) if dtype == F16 else (2.0 ** -20, 2.0 ** 40)
        v *= torch.where((block % 7 == 6) | (torch.arange(n) == n - 1), large, small)[:, None]
    elif kind == "mixed":
        sizes = torch.tensor([-60.0, -30.0, -9.0, 0.0, 0.0, 13.0, 40.0])
        v *= torch.exp2(sizes[torch.randint(0, 7, (n // 16 + 1,), generator=p.gen)])[block][:, None]
    elif kind == "outweighed":                         # every third block: values of 2^40 under scores some 28 (40 powers of two) lower
        k[..., 0] = torch.where(block % 3 == 1, -28.0, 0.0)
        q[..., 0] = dim ** 0.5
        v *= torch.where(block % 3 == 1, 2.0 ** 40, 1.0)[:, None]
    elif kind == "cliff":                              # beyond the first key tile scores 710 lower, 2^-1024, of values 2^60 apart
        k[..., 0] = torch.where(torch.arange(n) < 128, 0.0, -710.0)
        q[..., 0] = dim ** 0.5
        v *= torch.exp2(30.0 - 60 * (block % 2))[:, None]
    elif kind == "own block":                          # the last token's block holds nothing else: its tokens before it are zeros by its scale
        v[..., n - 1, :] *= 2.0 ** 40
    elif kind in ("rare", "first", "creeping"):
        # tokens of large values under weights of 2^-100 and less, whose blocks hold nothing else: now and then; in the first key tile; behind it ever larger ones, and
        # ordinary values at the end
        at = torch.arange(n)
        loud = {"rare": at % 53 == 31, "first": (at < 128) & (at % 16 == 5), "creeping": (at % 16 == 3) & (at >= 128) & (at < n - 200)}[kind]
        power = (at // 128 * 10).clamp(max=60).float() if kind == "creeping" else torch.full((n,), 40.0)
        k[..., 0] = torch.where(loud, -70.0 - power / 2, 0.0)
        q[..., 0] = dim ** 0.5
        v *= torch.where(loud, torch.exp2(power + 8), 1.0)[:, None]
    elif kind == "silent":                             # what takes nearly all weight has values of zero; what is left holds some 2^-12 of it
        k[..., 0] = torch.where(torch.arange(n) < 140, 8.0, 0.0)
        q[..., 0] = dim ** 0.5
        v[..., :140, :] = 0
    elif kind == "zeros":
        v *= (block % 40 >= 20).float()[:, None]
    else:                                              # products of -1e36: the first token is all that counts
        k = -torch.exp2(60.0 + (torch.arange(n) * 7 % 5))[None, None, :, None].expand(1, 1, -1, dim).contiguous()
        k[0, 0, 1:] *= 2
        q = torch.full((1, 2, tokens, dim), 2.0 ** 56).to(dtype)
        v *= (torch.where(block == 0, 1.0, torch.exp2(30.0 - 60 * (block % 2))) if kind == "far" else torch.exp2(2.0 * (block % 4)))[:, None]
    k, v = k.to(dtype), v.to(dtype)
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    want = p.plain.attend(0, q[0])[None]
    p.cache._prompt_work = 0
    got = p.cache.prefill_attention(0, q.to(DEV))
    close(got, want, dtype, weights=True)
    assert torch.equal(p.cache.prefill_attention(0, q.to(DEV)), got) and p.cache.kernel_status() == 0
    if kind in ("later", "zeros"):
        p.cache._prompt_work = 1 << 60
        close(p.cache.prefill_attention(0, q.to(DEV)), want, dtype)


def test_prompt_attention_of_rows_whose_reference_moves():
    """Scores that rise from key tile to key tile, beyond what weights in fp16 reach."""
    p = Pair(1, 1, 4, 64, BF16, pages=80)
    k = (torch.randn(1, 1, 700, 64, generator=p.gen) * 0.3 + (torch.arange(700) // 50 * 0.2)[None, None, :, None]).to(BF16)
    v = vectors(p.gen, 1, 1, 700, 64, BF16, large=False)
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    q = (torch.rand(1, 4, 300, 64, generator=p.gen) * torch.tensor([1.0, 3.0, -2.0, 0.1])[None, :, None, None]).to(BF16)
    p.cache._prompt_work = 0
    got = p.cache.prefill_attention(0, q.to(DEV))
    want = p.plain.attend(0, q[0])[None]
    # scores reach 130: 2^-22 of the largest product sums to 2e-5 * 130 / 20 in a weight; values of random sign as everywhere
    err = row_errors(got, want)
    assert float(err.max()) <= torch.finfo(BF16).eps / 2 + 2.0 ** -10 + 2e-4


def test_prompt_attention_of_sequences_of_different_lengths():
    p = Pair(3, 2, 4, 128, F16)
    p.append(30, batch=1)
    p.append(17, batch=2)
    p.append(40)
    p.check_prompt(40)
    p.check_prompt(3)                                  # any number of last tokens, not only the last chunk's


def test_weights_far_apart_and_rows_that_grow():
    """Scores that rise block by block, and one token that outweighs all others."""
    p = Pair(1, 1, 4, 64, F32, pages=80)
    k = torch.randn(1, 1, 1000, 64, generator=p.gen) * (1 + torch.arange(1000) / 100.0)[None, None, :, None]
    k[0, 0, 700] *= 30
    v = torch.randn(1, 1, 1000, 64, generator=p.gen) * torch.logspace(-6, 6, 1000)[None, None, torch.randperm(1000, generator=p.gen), None]
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    q = p.queries() * 0.05
    got = p.cache.decode_attention(0, q.to(DEV))
    want = p.plain.attend(0, q[0, :, None])[:, 0][None]
    # |s| reaches some 60 here, and the values' magnitudes differ by 2^40: what counts is the error relative to the weighted magnitudes
    size = p.plain.values(0, 1).abs()[0]
    w = torch.softmax(p.plain.values(0, 0)[0] @ q[0].double().T / 8, 0).T
    assert bool(((got.cpu().double() - want).abs()[0] <= 1e-4 * (w @ size)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim, past", [(64, 0), (128, 700)])
def test_scores_far_below_zero_are_scores(dtype, dim, past):
    """Products of -1e36: every one is finite in 32 bits, and what is seen is never a row without tokens. The keys' sizes are powers of two, so that a row's largest
    score stands alone by 1e35 and the answer is one token's value."""
    p = Pair(1, 1, 2, dim, dtype, pages=60)
    k = -torch.exp2(60.0 + (torch.arange(past + 20) * 7 % 5)).to(dtype)[None, None, :, None].expand(1, 1, -1, dim).contiguous()
    k[0, 0, 1:] *= 2                                   # the first token is the largest score of every row
    v = vectors(p.gen, 1, 1, past + 20, dim, dtype)
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    q = torch.full((1, 2, 20, dim), 2.0 ** 56).to(dtype)
    p.cache._prompt_work = 1 << 60
    want = p.plain.attend(0, q[0])[None]
    assert bool((want.norm(dim=-1) > 0).all())
    close(p.cache.decode_attention(0, q[:, :, -1].to(DEV)), want[:, :, -1], dtype)
    for work in (0, 1 << 60):
        p.cache._prompt_work = work
        close(p.cache.prefill_attention(0, q.to(DEV)), want, dtype, weights=work == 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("power", [16, 20, 23, 25, 27, 28, 29, 30, 31, 34, 45, 60])
def test_scores_of_any_size_choose_a_token(dtype, power):
    """Scores of 2^power: a product's rounding, 2^-24 of it, is many powers of two. Keys are random signs times a size each, queries some of the keys, so that a row's first
    two scores are further apart than any rounding and the answer is the first one's value."""
    p = Pair(1, 1, 4, 64, dtype, pages=60)
    n = 600
    k = torch.sign(torch.randn(1, 1, n, 64, generator=p.gen)) * (0.3 + 0.7 * torch.rand(1, 1, n, 1, generator=p.gen)) * 2.0 ** (power // 2)
    v = vectors(p.gen, 1, 1, n, 64, dtype, large=False)
    p.cache.append(0, k.to(dtype).to(DEV), v.to(DEV))
    p.plain.append(k.to(dtype), v)
    held = p.plain.values(0, 0)[0]
    at = torch.randint(0, n - 40, (1, 4, 40), generator=p.gen)
    q = (held[at] / 2.0 ** (power // 2) * 2.0 ** (power - power // 2) / 8).to(dtype)        # rows that ask for one of the tokens
    scores = torch.einsum("hqd,kd->hqk", q[0].double(), held) / 8
    top = scores.topk(2, -1).values
    clear = (top[..., 0] - top[..., 1]) > 2.0 ** -18 * top[..., 0].abs() + 64               # far beyond what 32 bits round
    assert float(clear.double().mean()) > 0.9
    want = p.plain.attend(0, q[0])[None]
    p.cache._prompt_work = 1 << 60
    last = p.cache.decode_attention(0, q[:, :, -1].to(DEV))
    close(last[:, clear[:, -1]], want[:, :, -1][:, clear[:, -1]], dtype)
    for work in (0, 1 << 60):
        p.cache._prompt_work = work
        got = p.cache.prefill_attention(0, q.to(DEV))
        close(got[:, clear], want[:, clear], dtype, weights=work == 0)
    assert p.cache.kernel_status() == 0


def test_queries_of_any_scale():
    for dtype, scale in ((BF16, 1e-30), (BF16, 1e4), (F32, 1e-35), (F32, 1e-3), (F16, 1e-4)):
        p = Pair(1, 2, 3, 64, dtype)
        p.append(50, scale=0.1 if scale > 1 else 1.0)
        q = (p.queries().float() * scale).to(dtype)
        if scale > 1:
            q = (q.float() * 1e-3).to(dtype)
        got = p.cache.decode_attention(0, q.to(DEV))
        close(got, p.plain.attend(0, q[0, :, None])[:, 0][None], dtype)
    p = Pair(1, 1, 2, 64, F32)
    p.append(50)
    zero = p.cache.decode_attention(0, torch.zeros(1, 2, 64, device=DEV))
    close(zero, p.plain.attend(0, torch.zeros(2, 1, 64))[:, 0][None], F32)


def test_other_strides_other_types_and_views():
    p = Pair(2, 2, 3, 64, BF16)
    k = vectors(p.gen, 2, 40, 2, 64, BF16).transpose(1, 2)          # [B, T, H, D] as a projection leaves it
    v = vectors(p.gen, 2, 2, 40, 2 * 64, BF16)[..., 64:]
    p.cache.append(0, k.to(DEV).transpose(1, 2).contiguous().transpose(1, 2), v.to(DEV))
    p.plain.append(k, v)
    p.check_pages()
    q = torch.randn(2, 40, 6, 64, generator=p.gen).to(BF16)
    on = q.to(DEV)
    for work in (0, 1 << 60):
        p.cache._prompt_work = work
        whole = p.cache.prefill_attention(0, on.transpose(1, 2))
        close(whole, torch.stack([p.plain.attend(b, q[b].transpose(0, 1)) for b in range(2)]), BF16, work == 0)
    one = p.cache.decode_attention(0, on.transpose(1, 2)[:, :, 7])
    assert torch.equal(one, p.cache.decode_attention(0, on[:, 7].contiguous()))
    odd = torch.zeros(2, 6, 68, dtype=BF16, device=DEV)
    odd[..., 3:67] = on[:, 7]
    assert torch.equal(p.cache.decode_attention(0, odd[..., 3:67]), one)
    double = p.cache.decode_attention(0, on[:, 7].double())          # a type that no kernel reads goes through the cache's own
    assert double.dtype == torch.float64 and torch.equal(double.to(BF16), one)
    mixed = p.cache.decode_attention(0, on[:, 7].float())            # queries need not be of the cache's type
    close(mixed, torch.stack([p.plain.attend(b, q[b, 7, :, None])[:, 0] for b in range(2)]), F32)


@pytest.mark.parametrize("k_type, v_type", [(F16, BF16), (BF16, F16), (F16, F32), (F32, BF16)])
def test_keys_and_values_of_different_types_keep_their_numbers(k_type, v_type):
    """Values of 1e6 beside keys in fp16, and keys of eleven bits beside values in bf16."""
    p = Pair(2, 2, 2, 64, BF16)
    for tokens in (19, 1):
        k, v = vectors(p.gen, 2, 2, tokens, 64, k_type), (vectors(p.gen, 2, 2, tokens, 64, F32) * (1.0 if v_type == F16 else 1e5)).to(v_type)
        p.cache.append(0, k.to(DEV), v.to(DEV))
        p.plain.append(k, v)
    p.check_pages()
    p.check_decode()


# ── blocks by score ──────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim, group", [(64, 1), (64, 16), (128, 4), (128, 5)])
@pytest.mark.parametrize("blocks, sinks, recent", [(4, 1, 2), (7, 0, 1), (9, 3, 5), (40, 1, 2)])
def test_chosen_blocks_are_the_best_ones(dtype, dim, group, blocks, sinks, recent):
    p = Pair(3, 2, group, dim, dtype, pages=100, seed=blocks)
    p.append(150)
    p.append(203, batch=2)
    p.append(60, batch=1)
    p.check_sparse(blocks, sinks, recent)


@pytest.mark.parametrize("tokens", [1, 16, 48, 63, 64, 65, 80, 81])
def test_short_sequences_are_read_whole(tokens):
    p = Pair(2, 1, 2, 64, F16, seed=tokens)
    p.append(tokens)
    chosen = p.check_sparse(4)
    assert chosen.shape == (2, 1, 4)
    q = p.queries().to(DEV)
    if tokens <= 64:
        assert torch.equal(p.cache.sparse_decode_attention(0, q, 4), p.cache.decode_attention(0, q))


def test_equal_scores_go_to_the_earlier_block():
    p = Pair(1, 2, 2, 64, F16, pages=64)
    k = vectors(p.gen, 1, 2, 16, 64, F16).repeat(1, 1, 50, 1)       # every block is the same
    p.cache.append(0, k.to(DEV), k.to(DEV))
    p.plain.append(k, k)
    assert p.check_sparse(9, 1, 2)[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 48, 49]
    p.cache.reset()
    p.plain = obytes.Cache(1, 2, 64)
    zeros = torch.zeros(1, 2, 700, 64, dtype=F16)
    p.cache.append(0, zeros.to(DEV), k[:, :, :700].to(DEV))
    p.plain.append(zeros, k[:, :, :700])
    assert p.check_sparse(6, 0, 1)[0, 1].tolist() == [0, 1, 2, 3, 4, 43]


@pytest.mark.parametrize("bad, blocks", [(30, 32), (29, 32), (28, 32), (100, 32), (509, 32), (40, 4), (300, 301)])
def test_more_blocks_without_a_number_than_there_is_room_for(bad, blocks):
    """One sequence of three has ``bad`` key blocks that are no numbers: the first of them are chosen, and the lists of the others are what they are without it."""
    p = Pair(3, 2, 2, 64, BF16, pages=1600, seed=bad)
    k, v = (vectors(p.gen, 3, 2, 16 * 512, 64, BF16) for _ in range(2))
    at = 16 * (1 + torch.randperm(509, generator=p.gen)[:bad])
    k[1, 1, at, 3] = torch.tensor([math.inf, -math.inf, math.nan], dtype=BF16)[torch.arange(bad) % 3]
    p.cache.append(0, k.to(DEV), v.to(DEV))
    p.plain.append(k, v)
    q = p.queries()
    got, chosen = p.cache.sparse_decode_attention(0, q.to(DEV), blocks, return_blocks=True)
    for b in range(3):
        want = p.plain.choose(b, q[b], blocks, 1, 2)
        assert torch.equal(chosen[b].cpu(), want), b
        out = p.plain.attend(b, q[b, :, None], want)[:, 0]
        if b == 1:
            assert bool(got[b, 2:].isnan().all())
            close(got[b, :2], out[:2], BF16)
        else:
            close(got[b], out, BF16)
    assert p.cache.kernel_status() == 0


@pytest.mark.parametrize("tokens, blocks", [(70000, 300), (16 * 4097, 33), (270000, 17)])
def test_choice_among_many_blocks(tokens, blocks):
    """More blocks than a small CTA, and than any CTA, keeps in registers; scores against the definition, vectorised."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    cache = ByteKVCache(num_layers=1, num_kv_heads=1, num_q_heads=2, head_dim=64, max_pages=tokens // 16 + 1, dtype=F16, device=DEV)
    k = torch.randn(1, 1, tokens, 64, generator=gen, device=DEV).to(F16)
    cache.append(0, k, k)
    q = torch.randn(1, 2, 64, generator=gen, device=DEV).to(F16)
    out, chosen = cache.sparse_decode_attention(0, q, blocks, return_blocks=True)
    codes, scales = cache.unpack_sequence(0, 0, 0)
    n = scales.shape[1]
    c = codes[0].double()[:16 * (tokens // 16)].view(-1, 16, 64)
    e = obytes.least_exponent(float(q.abs().max()), 2047)
    i = torch.round(q[0].double() * 2.0 ** -e)
    u = c.amax(1) @ i.clamp(min=0).sum(0) + c.amin(1) @ i.clamp(max=0).sum(0)
    score = u.float() * scales[0, :len(u)]
    score[0] = math.inf
    score = torch.cat([score, score.new_full((n - len(score),), 0.0)])
    score[n - 2:] = math.inf
    want = torch.sort(score, descending=True, stable=True).indices[:blocks].sort().values
    assert torch.equal(chosen[0, 0].long(), want)
    kk = (codes[0].double() * scales[0].double().repeat_interleave(16)[:tokens, None])
    at = (want[:, None] * 16 + torch.arange(16, device=DEV)).flatten()
    at = at[at < tokens]
    w = torch.softmax(q[0].double() @ kk[at].T / 8, -1)
    vc, vs = cache.unpack_sequence(0, 0, 1)
    close(out[0], (w @ (vc[0].double() * vs[0].double().repeat_interleave(16)[:tokens, None])[at]).cpu(), F16)


# ── as they are used ─────────────────────────────────────────────────────────────────────────────────────────

def test_a_prompt_in_chunks_then_single_tokens_on_several_layers():
    p = Pair(2, 2, 4, 128, BF16, layers=3, pages=40)
    plains = [p.plain] + [obytes.Cache(2, 2, 128) for _ in range(2)]
    for tokens in (33, 16, 1, 1, 7, 1):
        for layer in range(3):
            p.plain = plains[layer]
            p.append(tokens, layer=layer)
            q = p.queries(tokens)
            got = p.cache.prefill_attention(layer, q.to(DEV)) if tokens > 1 else p.cache.decode_attention(layer, q[:, :, 0].to(DEV))[:, :, None]
            close(got, torch.stack([p.plain.attend(b, q[b]) for b in range(2)]), BF16)
    for layer in range(3):
        p.plain = plains[layer]
        p.check_pages(layer)
    assert p.cache.seen_tokens == 59 and p.cache.get_seq_length() == 59


def test_update_returns_the_dense_cache():
    p = Pair(2, 2, 1, 64, F16)
    for tokens in (20, 1):
        k, v = (vectors(p.gen, 2, 2, tokens, 64, F16) for _ in range(2))
        dense = p.cache.update(k.to(DEV), v.to(DEV), 0)
        p.plain.append(k, v)
        for which in range(2):
            assert torch.equal(dense[which].cpu(), torch.stack([p.plain.values(b, which) for b in range(2)]).to(F16))


def test_captured_calls_on_another_stream_replay_on_new_inputs():
    p = Pair(2, 2, 4, 128, F16, pages=80)
    p.append(450)
    q = p.queries().to(DEV)
    p.cache.decode_attention(0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = p.cache.decode_attention(0, q)
        few, chosen = p.cache.sparse_decode_attention(0, q, 8, return_blocks=True)
        prompt = p.cache.prefill_attention(0, q[:, :, None].expand(-1, -1, 3, -1))
        p.cache._prompt_work = 0
        other = p.cache.prefill_attention(0, q[:, :, None].expand(-1, -1, 3, -1))
    for _ in range(3):
        new = p.queries()
        q.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        close(dense, torch.stack([p.plain.attend(b, new[b, :, None])[:, 0] for b in range(2)]), F16)
        for b in range(2):
            want = p.plain.choose(b, new[b], 8, 1, 2)
            assert torch.equal(chosen[b].cpu(), want)
            close(few[b], p.plain.attend(b, new[b, :, None], want)[:, 0], F16)
        want = torch.stack([p.plain.attend(b, new[b, :, None].expand(-1, 3, -1)) for b in range(2)])
        close(prompt, want, F16)
        close(other, want, F16, weights=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = p.cache.decode_attention(0, q)
    side.synchronize()
    # (a captured call is cut for the pool's size, this one for the sequences': the same sums in another order)
    close(again, torch.stack([p.plain.attend(b, new[b, :, None])[:, 0] for b in range(2)]), F16)
    assert p.cache.kernel_status() == 0


def test_a_replay_answers_for_the_lengths_that_the_sequences_have_by_then():
    """Captured over short sequences, replayed over long ones: other numbers of parts, of key tiles, and blocks that were not there."""
    p = Pair(2, 2, 4, 128, BF16, pages=1500)
    p.append(30)
    q, q3 = p.queries().to(DEV), p.queries(3).to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = p.cache.decode_attention(0, q)
        few, chosen = p.cache.sparse_decode_attention(0, q, 6, return_blocks=True)
        quiet = p.cache.sparse_decode_attention(0, q, 6)
        small = p.cache.prefill_attention(0, q3)
        p.cache._prompt_work = 0
        large = p.cache.prefill_attention(0, q3)
        with pytest.raises(RuntimeError, match="captured"):
            p.cache.append(0, torch.zeros(2, 2, 1, 128, dtype=BF16, device=DEV), torch.zeros(2, 2, 1, 128, dtype=BF16, device=DEV))
        with pytest.raises(RuntimeError, match="captured"):
            p.cache.crop(3)
    for more, batch in ((0, None), (1, None), (300, 1), (4000, None)):
        if more:
            p.append(more, batch=batch)
        new, new3 = p.queries(), p.queries(3)
        q.copy_(new), q3.copy_(new3)
        graph.replay()
        torch.cuda.synchronize()
        close(dense, torch.stack([p.plain.attend(b, new[b, :, None])[:, 0] for b in range(2)]), BF16)
        want = torch.stack([p.plain.attend(b, new3[b]) for b in range(2)])
        close(small, want, BF16)
        close(large, want, BF16, weights=True)
        for b in range(2):
            blocks = p.plain.choose(b, new[b], 6, 1, 2)
            assert torch.equal(chosen[b].cpu(), blocks)
            close(few[b], p.plain.attend(b, new[b, :, None], blocks)[:, 0], BF16)
        assert torch.equal(quiet, few) and p.cache.kernel_status() == 0
    one = p.cache.decode_attention(0, q[:1])
    close(one, p.plain.attend(0, new[0, :, None])[:, 0][None], BF16)


def test_no_layer_appends_inside_a_capture():
    cache = ByteKVCache(num_layers=2, num_kv_heads=1, num_q_heads=1, head_dim=64, max_pages=4, dtype=F16, device=DEV)
    k = vectors(torch.Generator().manual_seed(4), 1, 1, 3, 64, F16).to(DEV)
    for layer in range(2):
        cache.append(layer, k, k)
    before = cache.kv_data.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        doubled = k * 2
        for layer in range(2):
            with pytest.raises(RuntimeError, match="captured"):
                cache.append(layer, doubled, doubled)
    graph.replay()
    assert torch.equal(cache.kv_data, before) and cache.get_seq_length() == 3


def test_a_reset_is_not_captured():
    cache = ByteKVCache(num_layers=1, num_kv_heads=1, num_q_heads=1, max_pages=4, dtype=F16, device="cuda")
    k = vectors(torch.Generator().manual_seed(3), 1, 1, 20, 128, F16).to(DEV)
    cache.append(0, k, k)
    want = cache.decode_attention(0, k[:, :, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode_attention(0, k[:, :, 0])
        with pytest.raises(RuntimeError, match="captured"):
            cache.reset()
    graph.replay()
    assert cache.get_seq_length() == 20 and cache._device.index == k.get_device()
    # two sums, each 2e-5 off at most, and their roundings
    assert float(row_errors(out, want.double().cpu()).max()) <= torch.finfo(F16).eps + 4e-5


@pytest.mark.parametrize("batch", [1, 3])
def test_a_replay_behind_a_crop_or_a_reset_reads_what_is_left(batch):
    p = Pair(batch, 2, 4, 64, F16)
    p.append(40)
    q = p.queries().to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p.cache.decode_attention(0, q)
    p.cache.crop(21)
    p.plain.crop(21)
    graph.replay()
    close(out, torch.stack([p.plain.attend(b, q[b, :, None].cpu())[:, 0] for b in range(batch)]), F16)
    p.cache.reset()
    graph.replay()
    assert not bool(out.any())
    k = vectors(p.gen, batch, 2, 5, 64, F16).to(DEV)
    p.cache.append(0, k, k)
    graph.replay()
    torch.cuda.synchronize()
    fresh = obytes.Cache(batch, 2, 64)
    fresh.append(k.cpu(), k.cpu())
    close(out, torch.stack([fresh.attend(b, q[b, :, None].cpu())[:, 0] for b in range(batch)]), F16)
    assert p.cache.get_pages_used() == batch and p.cache.page_table_status() == 0 and p.cache.kernel_status() == 0


def test_a_larger_batch_leaves_the_tables_of_an_earlier_graph_alive():
    p = Pair(4, 1, 2, 64, F16)
    p.append(20, batch=1)
    q = torch.randn(1, 2, 64, generator=p.gen).to(F16).to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p.cache.decode_attention(0, q)
    want = p.plain.attend(0, q[0, :, None])[:, 0][None]
    k = vectors(p.gen, 4, 1, 3, 64, F16).to(DEV)
    p.cache.append(0, k, k)                            # new tables; the graph keeps to the lengths that it knew
    for _ in range(20):
        torch.zeros(1000, device=DEV)
    graph.replay()
    torch.cuda.synchronize()
    assert bool(out.isfinite().all()) and p.cache.kernel_status() == 0
    assert want.shape == out.shape


@pytest.mark.parametrize("known", [0, 1, 2])
def test_attention_captured_ahead_of_the_sequences_answers_once_they_are_there(known):
    """A capture for more sequences than have been appended leaves the cache as it was; the table is taken by the appends behind it."""
    p = Pair(4, 2, 2, 64, F16, pages=200)
    if known:
        p.append(21, batch=known)
    q = p.queries().to(DEV)
    table, lengths = p.cache._block_table, list(p.cache._seq_lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = p.cache.decode_attention(0, q)
        few, chosen = p.cache.sparse_decode_attention(0, q, 4, return_blocks=True)
    assert p.cache._block_table is table and p.cache._seq_lengths == lengths

    def check():
        graph.replay()
        torch.cuda.synchronize()
        for b in range(4):
            close(dense[b], p.plain.attend(b, q[b, :, None].cpu())[:, 0], F16)
            if p.plain.n[b]:
                want = p.plain.choose(b, q[b].cpu(), 4, 1, 2)
                assert torch.equal(chosen[b].cpu(), want)
                close(few[b], p.plain.attend(b, q[b, :, None].cpu(), want)[:, 0], F16)
        assert p.cache.kernel_status() == 0 and p.cache.page_table_status() == 0

    check()
    for tokens, batch in ((20, 2), (1, 2), (90, 4), (1, 3)):
        p.append(tokens, batch=batch)
        check()
        p.check_pages()
    p.check_decode()


def test_attention_captured_behind_a_crop_or_a_reset_replays_on_a_larger_table():
    """What these leave is in place before the capture: nothing that a replay would repeat on a table that has moved on."""
    p = Pair(4, 1, 2, 64, F16, pages=200)
    p.append(70, batch=2)
    p.cache.crop(50)
    p.plain.crop(50)
    q = p.queries().to(DEV)
    cropped, empty = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(cropped):
        first = p.cache.decode_attention(0, q[:2])
    cropped.replay()
    close(first, torch.stack([p.plain.attend(b, q[b, :, None].cpu())[:, 0] for b in range(2)]), F16)
    p.cache.reset()
    p.plain = obytes.Cache(4, 1, 64)
    with torch.cuda.graph(empty):
        second = p.cache.decode_attention(0, q)
    for tokens, batch in ((30, 1), (40, 4), (9, 2)):
        p.append(tokens, batch=batch)
        cropped.replay()
        empty.replay()
        torch.cuda.synchronize()
        want = torch.stack([p.plain.attend(b, q[b, :, None].cpu())[:, 0] for b in range(4)])
        close(first, want[:2], F16)
        close(second, want, F16)
        p.check_decode()                               # a replay has changed nothing that an eager call reads
        p.check_pages()


def test_a_table_that_does_not_fit_its_flat_arrays_is_not_captured():
    p = Pair(2, 1, 2, 64, F16)
    p.append(30)
    p.cache._free_sequence_pages(1)
    q = p.queries().to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        doubled = q * 2
        with pytest.raises(RuntimeError, match="before it is captured"):
            p.cache.decode_attention(0, q)
    graph.replay()
    assert torch.equal(doubled, q * 2)
    out = p.cache.decode_attention(0, q)
    close(out[0], p.plain.attend(0, q[0, :, None].cpu())[:, 0], F16)
    assert not bool(out[1].any())


def test_a_graph_from_before_the_table_grew_answers_for_what_the_sequences_hold():
    """Captured for two sequences, replayed with five: pages that are new by then, pages that were given back, and a table of one sequence again."""
    p = Pair(5, 2, 3, 64, BF16, pages=300)
    p.append(40, batch=2)
    q, q3 = p.queries()[:2].to(DEV), p.queries(3)[:2].to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = p.cache.decode_attention(0, q)
        few, chosen = p.cache.sparse_decode_attention(0, q, 4, return_blocks=True)
        prompt = p.cache.prefill_attention(0, q3)

    def check():
        graph.replay()
        torch.cuda.synchronize()
        for b in range(2):
            if p.plain.n[b] == 0:
                assert not bool(dense[b].any()) and not bool(few[b].any()) and not bool(prompt[b].any()) and bool((chosen[b] == -1).all())
                continue
            close(dense[b], p.plain.attend(b, q[b, :, None].cpu())[:, 0], BF16)
            close(prompt[b], p.plain.attend(b, q3[b].cpu()), BF16)
            want = p.plain.choose(b, q[b].cpu(), 4, 1, 2)
            assert torch.equal(chosen[b].cpu(), want)
            close(few[b], p.plain.attend(b, q[b, :, None].cpu(), want)[:, 0], BF16)
        assert p.cache.kernel_status() == 0 and p.cache.page_table_status() == 0

    check()
    p.append(33)                                       # five sequences: another block table
    held = [torch.full((1 << 18,), 7, dtype=torch.int32, device=DEV) for _ in range(8)]
    check()
    p.append(100, batch=1)
    check()
    p.append(5, batch=3)
    check()
    p.cache.crop(70)
    p.plain.crop(70)
    check()
    p.cache.reset()
    p.plain = obytes.Cache(5, 2, 64)
    check()
    p.append(50, batch=1)                              # the second sequence holds nothing
    check()
    p.append(9, batch=2)
    check()
    del held


def test_a_table_that_grows_on_another_stream_is_copied_before_its_memory_is_used_again():
    """The cache was made on the default stream, which goes on taking memory while the growth waits on a busy one."""
    p = Pair(3, 1, 2, 64, F16, pages=4096)
    p.append(200, batch=1)
    k, v = (vectors(p.gen, 3, 1, 20, 64, F16) for _ in range(2))
    on = k.to(DEV), v.to(DEV)
    torch.cuda.synchronize()
    held = len(p.cache._block_table)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                  # some 10 ms
        p.cache.append(0, *on)
    p.plain.append(k, v)
    for _ in range(4):                                 # of the old table's size
        torch.full((held, 4096), 77, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    assert len(p.cache._block_table) == 3
    p.check_pages()
    p.check_decode()


def test_two_caches_on_two_streams_at_once():
    pairs = [Pair(2, 2, 4, 128, BF16, pages=400, seed=21), Pair(1, 4, 3, 64, F16, pages=600, seed=22)]
    calls = []
    for p in pairs:
        p.append(2500)
        q, q3 = p.queries().to(DEV), p.queries(70).to(DEV)
        calls.append(lambda p=p, q=q, q3=q3: (p.cache.decode_attention(0, q), p.cache.prefill_attention(0, q3), p.cache.sparse_decode_attention(0, q, 20)))
        p.cache._prompt_work = 0
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pairs]
    got = [[], []]
    for _ in range(10):
        for f, stream, to in zip(calls, streams, got):
            with torch.cuda.stream(stream):
                to.append(f())
    torch.cuda.synchronize()
    for outs, first, p in zip(got, want, pairs):
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, first)) and p.cache.kernel_status() == 0


def test_pages_beyond_four_gigabytes():
    """The free stack hands out the last pages first: offsets of 6 GB and of 3 GB into the pool."""
    p = Pair(2, 8, 2, 128, F16, pages=200_000)
    assert p.cache.kv_data.numel() > 6 * 2 ** 30
    p.append(40)
    assert int(p.cache._block_table[0, 0]) > 199_000
    p.check_pages()
    p.check_decode()
    p.check_prompt(5)
    p.append(200)
    p.check_sparse(6)


def test_page_ids_outside_the_pool_are_reported_and_left_alone():
    """The kernels check every id against the pool: nothing is read or written there, the other sequences are answered."""
    p = Pair(3, 2, 2, 64, F16)
    p.append(40)
    before = p.cache.kv_data.clone()
    p.cache._device_meta(3)
    flat = p.cache._kv_page_indices
    good = flat.clone()
    for bad in (64, 1 << 30, -1, -(1 << 31)):
        flat[4] = bad                                  # sequence 1's second page
        q = p.queries()
        got = p.cache.decode_attention(0, q.to(DEV))
        for b in (0, 2):
            close(got[b], p.plain.attend(b, q[b, :, None])[:, 0], F16)
        p.cache.sparse_decode_attention(0, q.to(DEV), 2, 0, 1)
        p.cache.prefill_attention(0, q[:, :, None].expand(-1, -1, 9, -1).to(DEV))
        assert p.cache.kernel_status() == 2
        p.cache._workspace[:4].zero_()
        p.cache._prompt_work = 0
        got = p.cache.prefill_attention(0, q[:, :, None].to(DEV))
        for b in (0, 2):
            close(got[b], p.plain.attend(b, q[b, :, None]), F16, weights=True)
        assert p.cache.kernel_status() == 2
        p.cache._workspace[:4].zero_()
        assert p.cache[0][0].shape == (3, 2, 40, 64)
        assert torch.equal(p.cache.kv_data, before)
    flat.copy_(good)
    p.check_decode()


# ── HuggingFace models ───────────────────────────────────────────────────────────────────────────────────────

def _model(dtype):
    from transformers import MistralConfig, MistralForCausalLM

    torch.manual_seed(0)
    cfg = MistralConfig(vocab_size=512, hidden_size=384, intermediate_size=768, num_hidden_layers=2, num_attention_heads=6, num_key_value_heads=2,
                        head_dim=64, max_position_embeddings=512, rope_theta=1e6, tie_word_embeddings=False)
    return MistralForCausalLM(cfg).to(dtype).to(DEV).eval()


def _run(model, cache, prompts, forced):
    logits = []
    with torch.no_grad():
        for ids in prompts:
            logits.append(model(ids, past_key_values=cache, use_cache=True).logits.float().cpu())
        for tok in forced:
            logits.append(model(tok.reshape(-1, 1).to(DEV), past_key_values=cache, use_cache=True).logits[:, -1].float().cpu())
    return logits


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_model_on_the_8_bit_cache_answers_as_on_its_dense_keys_and_values(dtype):
    """Both routes use the same stored numbers; they differ by roundings of 16-bit attention and projections, a few eps of the logits each."""
    from leankv_b200.combined import optimize_model, reset_optimizations

    model = _model(dtype)
    gen = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 512, (2, n), generator=gen).to(DEV) for n in (45, 21)]
    forced = [torch.randint(0, 512, (2,), generator=gen) for _ in range(20)]
    _, dense = optimize_model(model, use_paged_cache=True, turboquant_bits=8, max_pages=64)
    assert isinstance(dense, ByteKVCache) and dense._dtype == dtype
    want = _run(model, dense, prompts, forced)
    for kw in (dict(), dict(fused_prefill=True), dict(fused_prefill=True, sparse_blocks=6)):
        _, cache = optimize_model(model, use_paged_cache=True, turboquant_bits=8, max_pages=64, fused_attention=True, **kw)
        got = _run(model, cache, prompts, forced)
        errs = [float((a - b).norm() / b.norm()) for a, b in zip(got, want)]
        assert max(errs) < 10 * torch.finfo(dtype).eps + 1e-3, (kw, errs)          # six blocks are all of 87 tokens
        assert cache.kernel_status() == 0 and cache.get_seq_length() == 45 + 21 + 20
        reset_optimizations(model)
        assert not cache.fused_decode and cache.sparse_blocks is None


def test_generate_reads_few_blocks():
    from leankv_b200.combined import optimize_model, reset_optimizations

    model = _model(F16)
    ids = torch.randint(0, 512, (1, 200), generator=torch.Generator().manual_seed(1)).to(DEV)
    _, cache = optimize_model(model, use_paged_cache=True, turboquant_bits=8, max_pages=64, fused_attention=True, fused_prefill=True, sparse_blocks=4)
    calls = []
    inner = cache.sparse_decode_attention
    cache.sparse_decode_attention = lambda layer, q, blocks: calls.append((layer, blocks)) or inner(layer, q, blocks)
    out = model.generate(ids, past_key_values=cache, max_new_tokens=9, do_sample=False, pad_token_id=0)
    assert out.shape == (1, 209) and calls == [(layer, 4) for _ in range(8) for layer in range(2)]
    reset_optimizations(model)
