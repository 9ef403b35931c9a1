"""The 8-bit paged cache on the CPU: its format's definition, the C ABI's checks, and the arguments that Python refuses."""

import copy
import ctypes
import math
import os
import pickle
import re

import pytest
import torch

from leankv_b200 import _native, combined
from leankv_b200.turboquant import byte_cache, hf_attention
from leankv_b200.turboquant.byte_cache import ByteKVCache, _is_prompt, _point
from leankv_b200.turboquant.paged_cache import PagedKVCache
from oracle import bytes as obytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "leankv_bytes.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(leankv_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(_native.BYTE_SIGNATURES)
    lib = _native.byte_lib()
    for n in names:
        assert hasattr(lib, n)
    assert lib.leankv_byte_chunk_bytes(128) == 4112 and lib.leankv_byte_chunk_bytes(64) == 2064
    assert lib.leankv_byte_bounds_bytes(128) == 272 and lib.leankv_byte_chunk_bytes(96) == 0


@pytest.mark.parametrize("most", [127, 2047])
def test_least_exponent_is_the_smallest_that_holds(most):
    gen = torch.Generator().manual_seed(0)
    numbers = [0.0, 1e-45, 2.0 ** -126, 2.0 ** 125, float(most), most * 2.0 ** -126, math.nextafter(float(most), 0), math.nextafter(float(most), 1e9)]
    numbers += [float(x) for x in torch.randn(200, generator=gen).abs() * torch.exp2(torch.randint(-100, 100, (200,), generator=gen).float())]
    for x in numbers:
        e = obytes.least_exponent(x, most)
        assert x <= math.ldexp(most, e) and e >= -126
        assert e == -126 or x > math.ldexp(most, e - 1)


def test_a_growing_scale_rounds_the_codes_again():
    block = obytes.Block(2)
    block.join(torch.tensor([[127.0, 3.0]], dtype=torch.float64))
    assert block.scale_exp == 0 and block.codes.tolist() == [[127.0, 3.0]]
    block.join(torch.tensor([[200.0, 0.0]], dtype=torch.float64))
    assert block.scale_exp == 1 and block.codes.tolist() == [[64.0, 2.0], [100.0, 0.0]]      # 63.5 and 1.5 to even
    block.join(torch.tensor([[math.inf, 0.0]], dtype=torch.float64))
    assert block.scale_exp is None and bool(block.values().isnan().all())


def _cpu_cache(**kw):
    return ByteKVCache(**{**dict(num_layers=2, num_kv_heads=2, num_q_heads=6, head_dim=64, max_pages=8, device="cpu"), **kw})


def test_shapes_that_the_kernels_do_not_have_are_refused():
    for bad in (dict(head_dim=96), dict(page_size=32), dict(bits=3), dict(num_q_heads=5), dict(num_q_heads=34), dict(num_q_heads=0),
                dict(dtype=torch.float64), dict(max_pages=0), dict(num_layers=0), dict(num_kv_heads=0)):
        with pytest.raises(RuntimeError):
            _cpu_cache(**bad)
    c = _cpu_cache()
    assert isinstance(c, PagedKVCache) and c.bytes_per_page() == 2 * (2064 + 144)
    assert c.kv_data.shape == (2, 8, 2, 2064) and c.get_pages_used() == 0 and c.get_seq_length() == 0
    for blocks, sinks, recent in ((2, 1, 2), (4, -1, 2), (4, 0, 0), (0, 0, 1)):
        with pytest.raises(RuntimeError, match="sparse"):
            c.check_blocks(blocks, sinks, recent)


def test_tensors_on_the_cpu_are_refused():
    c = _cpu_cache()
    k = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    for call in (lambda: c.append(0, k, k), lambda: c.update(k, k, 0), lambda: c.decode_attention(0, torch.zeros(1, 6, 64)),
                 lambda: c.prefill_attention(0, torch.zeros(1, 6, 3, 64)), lambda: c.sparse_decode_attention(0, torch.zeros(1, 6, 64), 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    assert c.get_seq_length() == 0 and c.get_pages_used() == 0


def test_rows_that_would_have_to_move_are_refused():
    cache = _cpu_cache()
    for call in (lambda: cache.reorder_cache(torch.tensor([0])), lambda: cache.batch_repeat_interleave(2), lambda: cache.batch_select_indices(torch.tensor([0]))):
        with pytest.raises(RuntimeError, match="places"):
            call()


def test_a_chunk_goes_to_the_kernel_that_takes_less():
    for pairs, group, dim, tokens, past, prompt in (
            (8, 4, 128, 64, 1000, False), (8, 4, 128, 128, 1000, True), (8, 4, 128, 8, 8000, False), (8, 4, 128, 16, 8000, True), (32, 4, 128, 4, 8000, False),
            (32, 4, 128, 16, 8000, True), (8, 4, 128, 64, 0, False), (8, 4, 128, 256, 0, True), (4, 3, 64, 128, 1000, False), (4, 3, 64, 64, 8000, True),
            (8, 1, 128, 1, 0, False), (1024 * 8, 16, 128, 4000, 100000, True)):
        assert _is_prompt(pairs, group, dim, tokens, -(-(past + tokens) // 16)) == prompt


def test_a_cache_is_not_copied():
    cache = _cpu_cache()
    for copied in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(RuntimeError, match="copied"):
            copied(cache)


def test_a_cache_is_not_made_inside_a_capture(monkeypatch):
    monkeypatch.setattr(byte_cache, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="inside a capture"):
        _cpu_cache(device="cuda:0")
    assert _cpu_cache().get_seq_length() == 0


def test_vectors_are_read_where_they_are_or_copied():
    d = _native.Vectors()
    x = torch.zeros(2, 3, 8, 64, dtype=torch.float16)
    assert _point(d, x) is x and (d.data, d.seq, d.head, d.token) == (x.data_ptr(), 3 * 8 * 64, 8 * 64, 64)
    view = torch.zeros(2, 8, 3, 64, dtype=torch.bfloat16).transpose(1, 2)
    assert _point(d, view) is view and (d.seq, d.head, d.token) == (8 * 3 * 64, 64, 3 * 64)
    one_token = view[:, :, 5]
    assert _point(d, one_token) is one_token and (d.data, d.seq, d.head) == (one_token.data_ptr(), 8 * 3 * 64, 64)
    for odd in (x.transpose(2, 3), torch.zeros(2, 3, 8, 68, dtype=torch.float16)[..., :64], x.reshape(-1)[4:-60].view(1, 1, -1, 64)[:, :, :2],
                torch.zeros(2, 3, 8, 66)[..., :64], torch.zeros(64 * 6 + 1, dtype=torch.float16)[1:].view(1, 1, 6, 64)):
        y = _point(d, odd)
        assert y is not odd and y.is_contiguous() and torch.equal(y, odd) and d.data == y.data_ptr() and y.data_ptr() % 16 == 0
    one = torch.zeros(1, 1, 1, 64, dtype=torch.float16).as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    assert _point(d, one) is one                       # strides of extents of one are not used


def test_structures_mirror_the_header(tmp_path):
    """Sizes and offsets of every field, from a compiled C program."""
    import subprocess

    kinds = {"leankv_byte_pool_t": _native.BytePool, "leankv_vectors_t": _native.Vectors, "leankv_byte_append_t": _native.ByteAppend,
             "leankv_byte_attn_t": _native.ByteAttn, "leankv_byte_select_t": _native.ByteSelect}
    lines = [f'printf("%zu {c}\\n", sizeof({c}));' for c in kinds]
    lines += [f'printf("%zu {c}.{f[0]}\\n", offsetof({c}, {f[0]}));' for c, t in kinds.items() for f in t._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "leankv_bytes.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = dict(reversed(line.split(" ")) for line in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, t in kinds.items():
        assert int(got[c]) == ctypes.sizeof(t)
        for f in t._fields_:
            assert int(got[f"{c}.{f[0]}"]) == getattr(t, f[0]).offset


def test_optimize_model_checks_what_sparse_blocks_needs():
    for kw in (dict(use_paged_cache=True, turboquant_bits=3, fused_attention=True), dict(use_paged_cache=True, turboquant_bits=8),
               dict(turboquant_bits=8, fused_attention=True)):
        with pytest.raises(ValueError, match="sparse_blocks"):
            combined.optimize_model(object(), sparse_blocks=32, **kw)
    with pytest.raises(RuntimeError, match="ByteKVCache"):
        hf_attention.enable_paged_attention(object(), PagedKVCache(num_layers=1, num_kv_heads=1, num_q_heads=4, max_pages=2, device="cpu"),
                                            sparse_blocks=8)
    with pytest.raises(RuntimeError, match="sparse"):
        hf_attention.enable_paged_attention(object(), _cpu_cache(), sparse_blocks=2)


def test_decode_steps_are_routed_to_the_chosen_blocks():
    """One-token steps go to ``sparse_decode_attention`` where the cache is set to it, and back when the plug-in is taken out."""
    asked = []

    class Cache:
        fused_decode, fused_prefill, sparse_blocks = True, False, 5

        def sparse_decode_attention(self, layer, q, blocks):
            asked.append((layer, tuple(q.shape), blocks))
            return q

        def decode_attention(self, layer, q):
            asked.append((layer, tuple(q.shape), None))
            return q

    class Module:
        layer_idx = 3
        _leankv_paged_cache = Cache()

    q = torch.zeros(2, 6, 1, 64)
    out, _ = hf_attention.paged_attention_forward(Module(), q, q, q, None)
    assert out.shape == (2, 1, 6, 64)
    Module._leankv_paged_cache.sparse_blocks = None
    hf_attention.paged_attention_forward(Module(), q, q, q, None)
    assert asked == [(3, (2, 6, 64), 5), (3, (2, 6, 64), None)]


def test_every_call_of_the_plug_in_sets_what_decode_steps_read():
    """Dense attention behind chosen blocks, on the same model or another, and a refused call that changes nothing."""
    from types import SimpleNamespace

    def model():
        return SimpleNamespace(model=SimpleNamespace(layers=[SimpleNamespace(self_attn=SimpleNamespace())]), config=SimpleNamespace(_attn_implementation="sdpa"))

    cache, first = _cpu_cache(), model()
    hf_attention.enable_paged_attention(first, cache, sparse_blocks=64)
    assert cache.sparse_blocks == 64
    hf_attention.enable_paged_attention(first, cache)
    assert cache.sparse_blocks is None
    hf_attention.enable_paged_attention(first, cache, sparse_blocks=8)
    with pytest.raises(RuntimeError, match="sparse"):
        hf_attention.enable_paged_attention(first, cache, sparse_blocks=1)
    assert cache.sparse_blocks == 8
    hf_attention.enable_paged_attention(model(), cache, fused_prefill=True)
    assert cache.sparse_blocks is None and cache.fused_prefill
    other = PagedKVCache(num_layers=1, num_kv_heads=1, num_q_heads=4, max_pages=2, device="cpu")
    hf_attention.enable_paged_attention(model(), other)
    assert not hasattr(other, "sparse_blocks")


# ── the C ABI: refused before any launch ─────────────────────────────────────────────────────────────────────

def _no_gpu():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where a check that stopped working cannot launch a kernel on them")


def _pool(**kw):
    f = dict(dim=128, kv_heads=2, n_pages=4, chunks=1 << 20, bounds=2 << 20)
    return _native.BytePool(**{**f, **kw})


def _vec(data=1 << 16, seq=4096, head=2048, token=128):
    return _native.Vectors(data, seq, head, token)


BAD_POOLS = [(dict(dim=96), -1), (dict(kv_heads=0), -1), (dict(n_pages=0), -1), (dict(chunks=None), -1), (dict(bounds=None), -1),
             (dict(chunks=(1 << 20) + 8), -2), (dict(bounds=(2 << 20) + 4), -2)]


def _append(lib, **kw):
    f = {**dict(pool=_pool(), dtype=0, batch=1, tokens=1, k=_vec(), v=_vec(), kv_indptr=64, kv_page_indices=64, kv_last_page_len=64), **kw}
    return lib.leankv_byte_append(ctypes.byref(_native.ByteAppend(**f)), None)


def test_append_and_unpack_check_their_arguments():
    _no_gpu()
    lib = _native.byte_lib()
    for bad, code in BAD_POOLS:
        assert _append(lib, pool=_pool(**bad)) == code
        assert lib.leankv_byte_unpack(ctypes.byref(_pool(**bad)), 0, 64, 64, 1, 1, 64, 64, 64, None) == code
    assert lib.leankv_byte_append(None, None) == -1 and lib.leankv_byte_unpack(None, 0, 64, 64, 1, 1, 64, 64, 64, None) == -1
    for kw, code in ((dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(batch=0), -1), (dict(tokens=0), -1), (dict(batch=1025), -6), (dict(kv_indptr=None), -1),
                     (dict(kv_page_indices=None), -1), (dict(kv_last_page_len=None), -1), (dict(k=_vec(data=None)), -1), (dict(v=_vec(data=24)), -2),
                     (dict(k=_vec(head=1028)), -2), (dict(v=_vec(seq=4), batch=2), -2), (dict(k=_vec(token=132), tokens=2), -2),
                     (dict(k=_vec(token=2 * 128 + 2), tokens=2, dtype=2), -2), (dict(batch=1024, tokens=2 ** 31 - 1), -6)):
        assert _append(lib, **kw) == code, kw
    f = lambda **kw: lib.leankv_byte_unpack(ctypes.byref(_pool()), *{**dict(dtype=0, k=64, v=64, B=1, T=1, ip=64, ids=64, last=64, st=None), **kw}.values())
    for kw, code in ((dict(dtype=5), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(T=-3), -1), (dict(B=1025), -6),
                     (dict(k=72), -2), (dict(v=40), -2), (dict(ip=None), -1), (dict(ids=None), -1), (dict(last=None), -1)):
        assert f(**kw) == code, kw


def test_dense_reads_check_where_they_write():
    lib = _native.byte_lib()
    f = lambda dtype, k, v: lib.leankv_byte_unpack(ctypes.byref(_pool()), dtype, k, v, 1, 1, 64, 64, 64, None)
    for dtype, good in ((_native.BYTES_F16, 16), (_native.BYTES_BF16, 16), (_native.BYTES_F32, 32)):
        assert f(dtype, 64 + good // 2, 64) == f(dtype, 64, 64 + good // 2) == -2


def test_attention_checks_its_arguments():
    _no_gpu()
    lib = _native.byte_lib()
    need = lib.leankv_byte_attn_workspace_bytes()

    def f(prompt=False, **kw):
        a = {**dict(pool=_pool(), dtype=0, batch=1, q_heads=8, tokens=1, q=_vec(), out=_vec(), scale=0.1, kv_indptr=64, kv_page_indices=64,
                    kv_last_page_len=64, max_pages_seq=4, total_pages=4, workspace=1 << 22, workspace_bytes=need), **kw}
        return (lib.leankv_byte_prompt_attn if prompt else lib.leankv_byte_attn)(ctypes.byref(_native.ByteAttn(**a)), None)

    for prompt in (False, True):
        for bad, code in BAD_POOLS:
            assert f(prompt, pool=_pool(**bad)) == code
        for kw, code in ((dict(dtype=3), -1), (dict(batch=0), -1), (dict(q_heads=0), -1), (dict(q_heads=7), -1), (dict(q_heads=34), -6), (dict(tokens=0), -1),
                         (dict(batch=1025), -6), (dict(kv_indptr=None), -1), (dict(kv_page_indices=None), -1), (dict(kv_last_page_len=None), -1),
                         (dict(max_pages_seq=-1), -1), (dict(total_pages=-1), -1), (dict(block_pages=64, n_blocks=0), -1),
                         (dict(block_pages=64, n_blocks=4, tokens=2), -1), (dict(workspace=None), -3), (dict(workspace_bytes=need - 1), -3),
                         (dict(workspace=(1 << 22) + 4), -2), (dict(q=_vec(data=None)), -1), (dict(out=_vec(data=None)), -1), (dict(q=_vec(data=4)), -2),
                         (dict(out=_vec(head=4)), -2), (dict(q=_vec(token=12), tokens=2), -2), (dict(tokens=1 << 30), -6)):
            assert f(prompt, **kw) == code, kw
    assert f(True, dtype=2) == -5 and f(True, scale=0.0) == -1 and f(True, scale=math.nan) == -1 and f(True, block_pages=64, n_blocks=4) == -1
    assert lib.leankv_byte_attn(None, None) == -1 and lib.leankv_byte_prompt_attn(None, None) == -1 and lib.leankv_byte_status(None, None) == -1


def test_select_checks_its_arguments():
    _no_gpu()
    lib = _native.byte_lib()

    def f(**kw):
        a = {**dict(pool=_pool(), dtype=0, batch=1, q_heads=8, q=_vec(), kv_indptr=64, kv_page_indices=64, max_pages_seq=40, n_blocks=8, sinks=1, recent=2,
                    blocks=64, block_pages=64, scores=64), **kw}
        return lib.leankv_byte_select(ctypes.byref(_native.ByteSelect(**a)), None)

    for bad, code in BAD_POOLS:
        assert f(pool=_pool(**bad)) == code
    assert lib.leankv_byte_select(None, None) == -1
    for kw, code in ((dict(dtype=9), -1), (dict(batch=0), -1), (dict(q_heads=3), -1), (dict(q_heads=64), -6), (dict(kv_indptr=None), -1),
                     (dict(kv_page_indices=None), -1), (dict(max_pages_seq=-1), -1), (dict(n_blocks=0), -1), (dict(sinks=-1), -1), (dict(recent=0), -1),
                     (dict(sinks=7), -1), (dict(blocks=None), -1), (dict(block_pages=None), -1), (dict(scores=None), -1), (dict(batch=1025), -6),
                     (dict(q=_vec(data=None)), -1), (dict(q=_vec(data=8)), -2), (dict(q=_vec(head=2)), -2)):
        assert f(**kw) == code, kw


def test_crop_checks_its_arguments():
    _no_gpu()
    lib = _native.lib()
    f = lambda **kw: lib.leankv_paged_table_crop(*{**dict(keep=1, B=1, n=64, table=64, pps=4, stack=64, top=64, size=4, status=64, st=None), **kw}.values())
    for kw, code in ((dict(keep=-1), -1), (dict(B=0), -1), (dict(B=1025), -6), (dict(pps=0), -1), (dict(size=0), -1), (dict(n=None), -1),
                     (dict(table=None), -1), (dict(stack=None), -1), (dict(top=None), -1), (dict(status=None), -1)):
        assert f(**kw) == code, kw
