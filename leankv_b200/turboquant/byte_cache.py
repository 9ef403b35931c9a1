"""Paged KV cache in 8 bits, with attention over all of it or over the blocks that score best.

The reference keeps fp16 pages (``leankv/turboquant/paged_cache.py``) or 3-bit codes (``leankv/turboquant/cache.py``); this cache stands
between the two. A block is the 16 tokens of a page, of one kv head, keys or values: codes ``rint(x * 2^-e)`` in -127 .. 127
and one scale 2^e, the smallest power of two that holds the block's largest magnitude. No rotation, no calibration; the error of a
number is at most half a step, 1/254 to 1/127 of the block's largest magnitude. A token that joins a block may raise its scale; the
codes that are there are then rounded once more. Powers of two make every rounding the same wherever it is done.

The page table, its kernels and the HF surface are those of ``PagedKVCache``. Beside it: head sizes 64 and 128, any group of up to 16 query
heads a kv head, keys, values and queries in fp16, bf16 or fp32, tensors of any strides of whole 16-byte pieces, ``crop``, and
``sparse_decode_attention``, which reads the blocks whose upper bound of the query's scores is largest.

    cache = ByteKVCache(num_layers=..., num_kv_heads=8, num_q_heads=32, dtype=torch.bfloat16, device="cuda")
    cache.append(layer, k, v)                                   # [B, Hkv, T, D]
    out = cache.prefill_attention(layer, q)                     # [B, Hq, T, D], the T tokens just appended
    out = cache.decode_attention(layer, q)                      # [B, Hq, D]
    out = cache.sparse_decode_attention(layer, q, blocks=128)   # the same, 128 blocks per kv head

A cache is used by one stream at a time: its pages, its page table and the workspace of its attention are one set. Attention may be captured into
a CUDA graph; a replay answers for the lengths that the sequences have by then, however many sequences there are.
Appends and ``crop`` are not captured: the host keeps the lengths, too.
"""

from __future__ import annotations

import ctypes
import functools
import math
from ctypes import byref

import torch

from .. import _native
from .paged_cache import PAGE, PagedKVCache

_TYPES = {torch.float16: _native.BYTES_F16, torch.bfloat16: _native.BYTES_BF16, torch.float32: _native.BYTES_F32}


def _point(v: _native.Vectors, t: torch.Tensor) -> torch.Tensor:
    """Fills ``v`` from ``t`` ([B, H, T, D] or [B, H, D]); returns the tensor that ``v`` points to: ``t`` where the kernels can read it, each
    vector contiguous and all of them from 16-byte boundaries on, else a copy."""
    strides, at = t.stride(), t.data_ptr()
    loose = 16 // t.element_size() - 1
    if len(strides) == 4:
        seq, head, token, one = strides
    else:
        (seq, head, one), token = strides, 0
    if one != 1 or at & 15 or (seq | head | token) & loose:
        # strides of extents of one are not used
        if one != 1 or at & 15 or any(s & loose and n > 1 for s, n in zip(strides, t.shape[:-1])):
            return _point(v, t.clone(memory_format=torch.contiguous_format))
    v.data, v.seq, v.head, v.token = at, seq, head, token
    return t


@functools.lru_cache(maxsize=4096)
def _is_prompt(pairs: int, group: int, dim: int, tokens: int, pages: int) -> bool:
    """Whether a chunk is taken by the prompt kernel, by what either kernel is expected to take (us). The one for few tokens reads the pages
    once for 16 (token, query head) rows: 6 and one for each 550 of them (head size 64: 5, 1000). The prompt kernel goes through tiles of 8 pages, 2 (1.6) each
    behind 8 (6.5), shared by as many CTAs as the device's 148 SMs hold; joining them is another 7 (5). Measured, few tokens' / prompt kernel, 8 kv heads of 4, head size 128: 64 tokens
    after 1000 20 / 24, 128 30 / 25; 8 after 8000 26 / 28, 16 35 / 29, 4 of four sequences 35 / 44, 16 83 / 44; 128 after none 9 / 10, 256 16 / 12."""
    few = 6 + pairs * -(-tokens * group // 16) * pages / 550 if dim == 128 else 5 + pairs * -(-tokens * group // 16) * pages / 1000
    units, tiles = pairs * -(-tokens // (2 * (128 // group))), -(-pages // 8)
    shares = max(1, min(148 // units, tiles // 4))
    if shares > 8:
        shares -= shares % 8
    steps = -(-tiles // shares) * -(-units // 148)
    prompt = 8 + 2 * steps + 7 * (shares > 1) if dim == 128 else 6.5 + 1.6 * steps + 5 * (shares > 1)
    return few > prompt


def _capturing() -> bool:
    return torch._C._cuda_isCurrentStreamCapturing()


class ByteKVCache(PagedKVCache):
    """Page pool of 8-bit keys and values + attention on it."""

    def __init__(self, num_layers: int = 32, num_kv_heads: int = 8, num_q_heads: int = 32, head_dim: int = 128, page_size: int = 16,
                 max_pages: int = 2048, dtype: torch.dtype = torch.float16, device=None, bits: int = 8):
        if head_dim not in (64, 128) or page_size != PAGE or bits != 8:
            raise RuntimeError("ByteKVCache kernels need head_dim 64 or 128, page_size=16, bits=8")
        if num_layers < 1 or max_pages < 1 or num_kv_heads < 1 or num_q_heads % num_kv_heads or \
                not 1 <= num_q_heads // num_kv_heads <= _native.BYTES_MAX_GROUP:
            raise RuntimeError("ByteKVCache needs layers, pages and 1 to 16 query heads per kv head")
        if dtype not in _TYPES:
            raise RuntimeError("ByteKVCache returns float16, bfloat16 or float32")
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.num_q_heads = num_q_heads
        self.head_dim = head_dim
        self.page_size = page_size
        self.max_pages = max_pages
        self.bits = bits
        self._dtype = dtype
        self._device = torch.device(device) if device is not None else torch.device("cuda")
        if self._device.type == "cuda" and _capturing():
            raise RuntimeError("ByteKVCache: a cache cannot be made inside a capture: its page table would be cleared by every replay")
        if self._device.type == "cuda" and self._device.index is None:
            self._device = torch.device("cuda", torch.cuda.current_device())       # whichever device is current in later calls
        self._seen_tokens = 0

        # [layer][page][kv head][keys | values | scales] and [layer][page][kv head][largest | smallest key code | scale]
        self._chunk, self._bound = 32 * head_dim + 16, 2 * head_dim + 16
        zeros = lambda n: torch.zeros(num_layers, max_pages, num_kv_heads, n, dtype=torch.uint8, device=self._device)
        self.kv_data, self.bounds = zeros(self._chunk), zeros(self._bound)
        self._seq_lengths: list[int] = []
        self._batch_size = 0
        self._free_count = max_pages
        self.fused_decode = False
        self.fused_prefill = False
        self.sparse_blocks = None             # set by hf_attention.enable_paged_attention
        # not on first use: a call that is being captured would record the clearing instead of doing it
        size = _native.byte_lib().leankv_byte_attn_workspace_bytes() if self._device.type == "cuda" else 0
        self._workspace = torch.zeros(size, dtype=torch.uint8, device=self._device)
        # None: by the rule above; else the pages read by 16 (token, query head) rows at a time from which a chunk goes to the prompt kernel
        self._prompt_work = None
        # the calls' arguments, one set for each layer: a call fills in what changes
        self._args, self._pools = [], []
        for i in range(num_layers):
            pool = _native.BytePool(head_dim, num_kv_heads, max_pages, self.kv_data[i].data_ptr(), self.bounds[i].data_ptr())
            self._pools.append(byref(pool))
            append = _native.ByteAppend(pool=pool)
            attn = _native.ByteAttn(pool=pool, q_heads=num_q_heads, scale=1.0 / math.sqrt(head_dim), workspace=self._workspace.data_ptr(),
                                    workspace_bytes=size)
            select = _native.ByteSelect(pool=pool, q_heads=num_q_heads)
            # (arguments, what a call passes, its tensors)
            self._args.append(((append, byref(append), append.k, append.v), (attn, byref(attn), attn.q, attn.out), (select, byref(select), select.q)))
        self._device_index = self.kv_data.get_device()
        self._lib, self._table_lib = _native.byte_lib(), _native.lib()
        self._alloc_tables(0)

    def _alloc_tables(self, batch_cap: int):
        """Room for the pages of ``batch_cap`` sequences. Only the block table ever moves: lengths and flat arrays, which the kernels of a captured call
        read, have their place for as many sequences as a call may have (16 KB)."""
        dev, i32 = self._device, torch.int32
        table = getattr(self, "_block_table", None)
        self._batch_cap = max(batch_cap, 1)
        self._pps_cap = self.max_pages                       # a single sequence may take the whole pool
        if table is None:
            most = _native.BYTES_MAX_BATCH
            # one allocation, each array from a 16-byte boundary on; zeros as far as the free stack
            sizes = [most, most + 1, most, most, self.max_pages, 1, self.max_pages, 1]
            padded = [-(-n // 4) * 4 for n in sizes]
            store = torch.empty(sum(padded), dtype=i32, device=dev)
            (self._seq_len_dev, self._kv_indptr, self._kv_last, self._start_dev, self._kv_page_indices, self._status, self._free_stack,
             self._free_top) = (v[:n] for v, n in zip(store.split(padded), sizes))
            self._begin_args = (ctypes.c_void_p(store.data_ptr()), sum(padded[:6]), self.max_pages, sum(padded[:7]))
            self._begin(store)
            self._meta_batch = 0                             # sequences that the flat arrays were built for; -1: they are not the table's
            for args in self._args:
                for a in args:
                    a[0].kv_indptr, a[0].kv_page_indices = self._kv_indptr.data_ptr(), self._kv_page_indices.data_ptr()
                args[0][0].kv_last_page_len = args[1][0].kv_last_page_len = self._kv_last.data_ptr()
        # only places of pages that a sequence holds are read
        self._block_table = torch.empty(self._batch_cap, self._pps_cap, dtype=i32, device=dev)
        if table is not None:
            self._block_table[:len(table)] = table
            if table.is_cuda:                                # it may be of another stream than the copy's
                table.record_stream(torch.cuda.current_stream(dev))
        at = lambda t: ctypes.c_void_p(t.data_ptr())      # converted once, not at every call
        self._step_args = (at(self._seq_len_dev), at(self._block_table), ctypes.c_int(self._pps_cap), at(self._free_stack), at(self._free_top),
                           at(self._kv_indptr), at(self._kv_page_indices), at(self._kv_last), at(self._start_dev), at(self._status))

    def _begin(self, store=None):
        """No sequences: every page is free, lengths and flat arrays are zeros, so that a sequence behind the last one of a table has no pages (or
        fewer, where ``kv_indptr`` falls back to zero: none as well)."""
        if self._device.type != "cuda":
            store[:self._begin_args[1]].zero_()
            torch.arange(self.max_pages, out=self._free_stack)
            self._free_top.fill_(self.max_pages)
            return
        with _native.on_device(self._device):
            rc = self._table_lib.leankv_paged_table_begin(*self._begin_args, _native.current_stream())
        if rc:
            _native.check(rc, "leankv_paged_table_begin")

    def _table_step(self, t_new: int, batch: int):
        with _native.on_device(self._device):
            self._step(t_new, batch, _native.current_stream())

    def _step(self, t_new: int, batch: int, stream: int):
        rc = self._table_lib.leankv_paged_table_step(t_new, batch, *self._step_args, stream)
        if rc:
            _native.check(rc, "leankv_paged_table_step")
        self._meta_batch = batch

    def _device_meta(self, batch_size: int):
        """(kv_indptr, kv_page_indices, kv_last_page_len) int32 on the device, for all known sequences: the first ones' part is the same
        for any smaller batch. A capture finds them as they are, with no pages for sequences that nobody knows yet: it neither takes
        memory for the table, which would be the graph's, nor records steps, which later replays would take on a table that has moved on."""
        if self._meta_batch < batch_size:
            if self._device.type != "cuda" or not _capturing():
                self._ensure_batch_size(batch_size)
                self._table_step(0, len(self._seq_lengths))
            elif self._meta_batch < 0:
                raise RuntimeError("ByteKVCache: the page table has changed: call the attention once before it is captured")
        return self._kv_indptr, self._kv_page_indices, self._kv_last

    # ── arguments ──────────────────────────────────────────────────────

    def _layer(self, layer_idx: int) -> tuple:
        if not 0 <= layer_idx < self.num_layers:
            raise RuntimeError(f"ByteKVCache has layers 0 .. {self.num_layers - 1}, not {layer_idx}")
        return self._args[layer_idx]

    def _typed(self, t: torch.Tensor, name: str, heads: int, batch=None, tokens=None, dims: int = 4) -> torch.Tensor:
        """``t`` ([batch, heads, tokens, head_dim], or without the tokens) after the checks that every call makes; a type that the
        kernels do not read becomes the cache's own."""
        shape = t.shape
        if (not t.is_cuda or t.get_device() != self._device_index or len(shape) != dims or shape[1] != heads or shape[-1] != self.head_dim
                or not 1 <= shape[0] <= _native.BYTES_MAX_BATCH or (batch is not None and (shape[0] != batch or shape[2] != tokens))):
            _native.require_cuda(t, name)
            if t.get_device() != self._device_index:
                raise RuntimeError(f"{name} is on {t.device}, the cache on {self.kv_data.device}")
            want = [f"1 .. {_native.BYTES_MAX_BATCH}" if batch is None else batch, heads, "*" if tokens is None else tokens, self.head_dim]
            raise RuntimeError(f"{name} must be {want if dims == 4 else want[:2] + want[3:]}, not {list(shape)}")
        return t if t.dtype in _TYPES else t.to(self._dtype)

    def check_blocks(self, blocks: int, sinks: int = 1, recent: int = 2) -> None:
        if sinks < 0 or recent < 1 or blocks < sinks + recent:
            raise RuntimeError("sparse attention needs recent >= 1, sinks >= 0 and blocks >= sinks + recent")

    def _most_pages(self, batch: int) -> int:
        """Of any of the first sequences; of any there may be where a graph is captured, whose replays meet longer ones."""
        if _capturing():
            return self.max_pages
        return -(-max(self._seq_lengths[:batch]) // PAGE)

    # ── appends ────────────────────────────────────────────────────────

    def append(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor):
        """Codes of ``[B, Hkv, T_new, D]`` K/V of one layer go into the pages of the first B sequences. Layer 0 advances the page table
        that all layers share; the other layers' tokens of the same step follow it."""
        k = self._typed(key_states, "key_states", self.num_kv_heads)
        batch, t_new = k.shape[0], k.shape[2]
        v = self._typed(value_states, "value_states", self.num_kv_heads, batch, t_new)
        (args, call, kp, vp), _, _ = self._layer(layer_idx)
        if k.dtype != v.dtype:                # a type that holds the numbers of both: a cast of one to the other's would round it, or lose its range
            k, v = k.float(), v.float()
        if t_new == 0:
            return
        if _capturing():
            raise RuntimeError("ByteKVCache: append goes by lengths that the host keeps, too, and cannot be captured")
        known = self._seq_lengths
        if layer_idx == 0:
            lengths = known[:batch] + [0] * (batch - len(known))
            if t_new == 1:
                need = [n % PAGE for n in lengths].count(0)
            else:
                need = sum([-(-(n + t_new) // PAGE) - -(-n // PAGE) for n in lengths])
            if need > self._free_count:
                raise RuntimeError(f"ByteKVCache: out of pages ({self.max_pages} used). "
                                   f"Increase max_pages or reduce batch/sequence length.")
            if len(known) < batch:
                self._ensure_batch_size(batch)
        elif len(known) < batch or min(known[:batch]) < t_new:
            raise RuntimeError("ByteKVCache: layer 0 has not appended these tokens yet")
        elif self._meta_batch < batch:
            self._device_meta(batch)
        args.dtype, args.batch, args.tokens = _TYPES[k.dtype], batch, t_new
        k, v = _point(kp, k), _point(vp, v)
        with _native.on_device(self._device):
            stream = _native.current_stream()
            if layer_idx == 0:
                self._step(t_new, batch, stream)
                self._seen_tokens += t_new
                self._free_count -= need
                known[:batch] = [n + t_new for n in lengths]
                if batch < len(known):
                    self._step(0, len(known), stream)
            rc = self._lib.leankv_byte_append(call, stream)
        if rc:
            _native.check(rc, "leankv_byte_append", self._lib)

    def _gather_kv(self, layer_idx: int, batch_size: int):
        """Dense ``[B, Hkv, max_seq, D]`` K and V in the cache's type (zeros behind a sequence's last token)."""
        self._layer(layer_idx)
        lengths = self._seq_lengths[:batch_size]
        max_seq = max(lengths) if lengths else 0
        shape = (batch_size, self.num_kv_heads, max_seq, self.head_dim)
        keys = torch.empty(shape, dtype=self._dtype, device=self._device)
        values = torch.empty_like(keys)
        if batch_size and max_seq:
            if self._meta_batch < batch_size:
                self._device_meta(batch_size)
            with _native.on_device(self._device):
                rc = self._lib.leankv_byte_unpack(self._pools[layer_idx], _TYPES[self._dtype], keys.data_ptr(), values.data_ptr(), batch_size, max_seq,
                                                  *self._step_args[5:8], _native.current_stream())
            if rc:
                _native.check(rc, "leankv_byte_unpack", self._lib)
        return keys, values

    def unpack_sequence(self, layer_idx: int, batch_idx: int, which: int):
        """Codes (int8 ``[Hkv, T, D]``) and scales (fp32 ``[Hkv, blocks]``) of one sequence's keys (0) or values (1)."""
        self._layer(layer_idx)
        t, d, h = self._seq_lengths[batch_idx], self.head_dim, self.num_kv_heads
        n = -(-t // PAGE)
        c = self.kv_data[layer_idx][self._block_table[batch_idx, :n].long()].transpose(0, 1).reshape(h, n, -1)
        scales = c[..., 32 * d:32 * d + 8].contiguous().view(torch.float32)[..., which]
        c = c[..., 16 * d * which:16 * d * (which + 1)]
        if which == 0:
            c = c.reshape(h, n, d // 64, PAGE, 64).permute(0, 1, 3, 2, 4).reshape(h, n * PAGE, d)
        else:      # [part][g][t][word][token of four]: channel 32 part + 8 word + g, token 2 t + {0, 1, 8, 9}
            c = c.reshape(h, n, d // 32, 8, 4, 4, 2, 2).permute(0, 1, 6, 4, 7, 2, 5, 3).reshape(h, n * PAGE, d)
        return (c[:, :t].to(torch.int16) - 128).to(torch.int8), scales

    # ── attention ──────────────────────────────────────────────────────

    def _attend(self, layer_idx: int, q: torch.Tensor, out: torch.Tensor, tokens: int, pages: int, lists=None, n_lists: int = 0,
                prompt: bool = False) -> None:
        """``q`` and ``out`` [B, Hq, (T,) D]: the last ``tokens`` tokens of each sequence over the pages."""
        a, call, qp, op = self._layer(layer_idx)[1]
        batch = q.shape[0]
        if self._meta_batch < batch:
            self._device_meta(batch)
        a.dtype, a.batch, a.tokens, a.max_pages_seq = _TYPES[q.dtype], batch, tokens, pages
        a.total_pages = self.max_pages if pages == self.max_pages else self.max_pages - self._free_count
        a.block_pages, a.n_blocks = lists, n_lists
        q = _point(qp, q)
        _point(op, out)
        with _native.on_device(self._device):
            rc = (self._lib.leankv_byte_prompt_attn if prompt else self._lib.leankv_byte_attn)(call, _native.current_stream())
        if rc:
            _native.check(rc, "leankv_byte_attn", self._lib)

    def _answer(self, q: torch.Tensor) -> torch.Tensor:
        """Room for a one-token answer."""
        if len(self._seq_lengths) < q.shape[0] and not _capturing():
            self._ensure_batch_size(q.shape[0])
        return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)

    def decode_attention(self, layer_idx: int, query: torch.Tensor) -> torch.Tensor:
        """``softmax(q K^T / sqrt(d)) V`` over every stored token of each sequence; query/out ``[B, Hq, D]``."""
        q = self._typed(query, "query", self.num_q_heads, dims=3)
        out = self._answer(q)
        self._attend(layer_idx, q, out, 1, self._most_pages(q.shape[0]))
        return out if out.dtype == query.dtype else out.to(query.dtype)

    def sparse_decode_attention(self, layer_idx: int, query: torch.Tensor, blocks: int, sinks: int = 1, recent: int = 2,
                                return_blocks: bool = False):
        """``decode_attention`` that reads at most ``blocks`` blocks (of 16 tokens) per sequence and kv head: the first ``sinks``, the last
        ``recent``, and those with the largest upper bound of the group's summed scores (from the largest and smallest key code of
        each channel; ties to the earlier block). With ``return_blocks`` also their numbers, ascending and then -1, int32
        ``[B, Hkv, blocks]``. A sequence of no more than ``blocks`` blocks is read whole."""
        q = self._typed(query, "query", self.num_q_heads, dims=3)
        self.check_blocks(blocks, sinks, recent)
        batch, heads = q.shape[0], self.num_kv_heads
        out = self._answer(q)
        pages = self._most_pages(batch)
        if pages <= blocks and not return_blocks:
            self._attend(layer_idx, q, out, 1, pages)
        else:
            a, call, qp = self._layer(layer_idx)[2]
            if self._meta_batch < batch:
                self._device_meta(batch)
            n = batch * heads * blocks
            words = torch.empty(2 * n + batch * heads * pages, dtype=torch.int32, device=q.device)      # numbers, page ids, scores
            at = words.data_ptr()
            a.dtype, a.batch = _TYPES[q.dtype], batch
            q = _point(qp, q)
            a.max_pages_seq, a.n_blocks, a.sinks, a.recent = pages, blocks, sinks, recent
            a.blocks, a.block_pages, a.scores = at, at + 4 * n, at + 8 * n
            with _native.on_device(self._device):
                rc = self._lib.leankv_byte_select(call, _native.current_stream())
            if rc:
                _native.check(rc, "leankv_byte_select", self._lib)
            self._attend(layer_idx, q, out, 1, pages, at + 4 * n, blocks)
        out = out if out.dtype == query.dtype else out.to(query.dtype)
        return (out, words[:n].view(batch, heads, blocks)) if return_blocks else out

    def prefill_attention(self, layer_idx: int, query: torch.Tensor) -> torch.Tensor:
        """Causal attention of the last T tokens of every sequence (the chunk that ``append`` has just added) over everything up to
        each: query/out ``[B, Hq, T, D]``."""
        q = self._typed(query, "query", self.num_q_heads)
        batch, _, t_new, _ = q.shape
        if len(self._seq_lengths) < batch or min(self._seq_lengths[:batch]) < t_new:
            raise RuntimeError("prefill_attention: the chunk has not been appended to this sequence")
        out = torch.empty(batch, t_new, self.num_q_heads, self.head_dim, dtype=q.dtype, device=q.device).transpose(1, 2)
        if t_new:
            group = self.num_q_heads // self.num_kv_heads
            pages = self._most_pages(batch)
            if q.dtype == torch.float32:
                prompt = False
            elif self._prompt_work is None:
                prompt = _is_prompt(batch * self.num_kv_heads, group, self.head_dim, t_new, pages)
            else:
                prompt = batch * self.num_kv_heads * -(-t_new * group // 16) * pages > self._prompt_work
            self._attend(layer_idx, q, out, t_new, pages, prompt=prompt)
        return out if out.dtype == query.dtype else out.to(query.dtype)

    def kernel_status(self) -> int:
        """Status word of the attention's bounded waits and page checks (0 = clean, bit 0: a wait ran out, bit 1: a page id outside
        the pool, bit 2: a table with more pages than the pool)."""
        val = ctypes.c_int(0)
        if self._workspace.is_cuda:
            with _native.on_device(self._device):
                _native.check(_native.byte_lib().leankv_byte_status(self._workspace.data_ptr(), byref(val)), "leankv_byte_status",
                              _native.byte_lib())
        return val.value

    # ── page table ─────────────────────────────────────────────────────

    def crop(self, max_length: int):
        """Cut every sequence back to at most ``max_length`` tokens (below zero: that many tokens fewer than the longest has), as after
        drafted tokens that were not accepted. The scale of a block that keeps some tokens stays as it is, a block that holds no number
        included."""
        if self._device.type == "cuda" and _capturing():
            raise RuntimeError("ByteKVCache: crop changes lengths that the host keeps, too, and cannot be captured")
        if max_length < 0:
            max_length = max(self.get_seq_length() + max_length, 0)
        batch = len(self._seq_lengths)
        if not batch or max(self._seq_lengths) <= max_length:
            return
        with _native.on_device(self._device):
            stream = _native.current_stream()
            rc = self._table_lib.leankv_paged_table_crop(max_length, batch, self._seq_len_dev.data_ptr(), self._block_table.data_ptr(),
                                                         self._pps_cap, self._free_stack.data_ptr(), self._free_top.data_ptr(),
                                                         self.max_pages, self._status.data_ptr(), stream)
            if rc:
                _native.check(rc, "leankv_paged_table_crop")
            self._step(0, batch, stream)      # a replay reads the flat arrays without a call of this class in between
        kept = -(-max_length // PAGE)
        for b, n in enumerate(self._seq_lengths):
            if n > max_length:
                self._free_count += -(-n // PAGE) - kept
                self._seq_lengths[b] = max_length
        self._seen_tokens = min(self._seen_tokens, max_length)

    def reset(self):
        """Forget every sequence. Pages need no clearing: only positions that have been written are read."""
        if self._device.type != "cuda":
            return super().reset()
        if _capturing():
            raise RuntimeError("ByteKVCache: reset changes lengths that the host keeps, too, and cannot be captured")
        self._begin()
        self._seq_lengths = []
        self._batch_size = 0
        self._seen_tokens = 0
        self._free_count = self.max_pages
        self._meta_batch = 0

    def _one_row_each(self, *args):
        raise RuntimeError("ByteKVCache keeps its sequences in their places: no beams, repeated or chosen rows")

    batch_repeat_interleave = batch_select_indices = reorder_cache = _one_row_each

    def _not_copied(self, *args):
        raise RuntimeError("ByteKVCache cannot be copied: its page table lies on the device")

    __copy__ = __deepcopy__ = __reduce_ex__ = _not_copied

    # ── diagnostics ────────────────────────────────────────────────────

    def bytes_per_page(self) -> int:
        """Bytes one page occupies in one layer (K and V, all kv heads, with the blocks' bounds)."""
        return self.num_kv_heads * (self._chunk + self._bound)

    def get_total_pool_mb(self) -> float:
        return (self.kv_data.numel() + self.bounds.numel()) / 1e6
