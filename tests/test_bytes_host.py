"""The 8-bit paged cache on the CPU: its format's definition, the C ABI's checks, and the arguments that Python refuses."""

import ctypes
import math
import os
import re

import pytest
import torch

from leankv_b200 import _native, combined
from leankv_b200.turboquant import hf_attention
from leankv_b200.turboquant.byte_cache import ByteKVCache, _vectors
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


def test_vectors_are_read_where_they_are_or_copied():
    x = torch.zeros(2, 3, 8, 64, dtype=torch.float16)
    d, y = _vectors(x)
    assert y is x and (d.seq, d.head, d.token) == (3 * 8 * 64, 8 * 64, 64)
    view = torch.zeros(2, 8, 3, 64, dtype=torch.bfloat16).transpose(1, 2)
    d, y = _vectors(view)
    assert y is view and (d.seq, d.head, d.token) == (8 * 3 * 64, 64, 3 * 64)
    for odd in (x.transpose(2, 3), torch.zeros(2, 3, 8, 68, dtype=torch.float16)[..., :64], x.reshape(-1)[4:-60].view(1, 1, -1, 64)[:, :, :2],
                torch.zeros(2, 3, 8, 66)[..., :64]):
        d, y = _vectors(odd)
        assert y.is_contiguous() and torch.equal(y, odd) and y.data_ptr() % 16 == 0
    one = torch.zeros(1, 1, 1, 64, dtype=torch.float16).as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    assert _vectors(one)[1] is one                     # strides of extents of one are not used


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


def _append(lib, pool=None, dtype=0, k=None, v=None, B=1, T=1, indptr=64, ids=64, last=64):
    return lib.leankv_byte_append(ctypes.byref(pool or _pool()), dtype, ctypes.byref(k or _vec()), ctypes.byref(v or _vec()), B, T, indptr, ids, last, None)


def test_append_and_unpack_check_their_arguments():
    _no_gpu()
    lib = _native.byte_lib()
    for bad, code in BAD_POOLS:
        assert _append(lib, _pool(**bad)) == code
        assert lib.leankv_byte_unpack(ctypes.byref(_pool(**bad)), 0, 64, 64, 1, 1, 64, 64, 64, None) == code
    assert lib.leankv_byte_append(None, 0, ctypes.byref(_vec()), ctypes.byref(_vec()), 1, 1, 64, 64, 64, None) == -1
    for kw, code in ((dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(B=1025), -6), (dict(indptr=None), -1),
                     (dict(ids=None), -1), (dict(last=None), -1), (dict(k=_vec(data=None)), -1), (dict(v=_vec(data=24)), -2),
                     (dict(k=_vec(head=1028)), -2), (dict(v=_vec(seq=4), B=2), -2), (dict(k=_vec(token=132), T=2), -2),
                     (dict(k=_vec(token=2 * 128 + 2), T=2, dtype=2), -2), (dict(B=1024, T=2 ** 31 - 1), -6)):
        assert _append(lib, **kw) == code, kw
    f = lambda **kw: lib.leankv_byte_unpack(ctypes.byref(_pool()), *{**dict(dtype=0, k=64, v=64, B=1, T=1, ip=64, ids=64, last=64, st=None), **kw}.values())
    for kw, code in ((dict(dtype=5), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(B=0), -1), (dict(T=0), -1), (dict(T=-3), -1), (dict(B=1025), -6),
                     (dict(k=72), -2), (dict(v=40), -2), (dict(ip=None), -1), (dict(ids=None), -1), (dict(last=None), -1)):
        assert f(**kw) == code, kw


def test_attention_checks_its_arguments():
    _no_gpu()
    lib = _native.byte_lib()
    need = lib.leankv_byte_attn_workspace_bytes()

    def f(pool=None, q=None, out=None, **kw):
        a = {**dict(B=1, heads=8, tokens=1, scale=0.1, ip=64, ids=64, last=64, pages=4, total=4, lists=None, n=0, ws=1 << 22, bytes=need, st=None), **kw}
        dtype, prompt = a.pop("dtype", 0), a.pop("prompt", False)
        if prompt:
            del a["total"], a["lists"], a["n"]
            return lib.leankv_byte_prompt_attn(ctypes.byref(pool or _pool()), dtype, ctypes.byref(q or _vec()), ctypes.byref(out or _vec()), *a.values())
        return lib.leankv_byte_attn(ctypes.byref(pool or _pool()), dtype, ctypes.byref(q or _vec()), ctypes.byref(out or _vec()), *a.values())

    for bad, code in BAD_POOLS:
        assert f(_pool(**bad)) == code and f(_pool(**bad), prompt=True) == code
    for kw, code in ((dict(dtype=3), -1), (dict(B=0), -1), (dict(heads=0), -1), (dict(heads=7), -1), (dict(heads=34), -6), (dict(tokens=0), -1),
                     (dict(B=1025), -6), (dict(ip=None), -1), (dict(ids=None), -1), (dict(last=None), -1), (dict(pages=-1), -1), (dict(total=-1), -1),
                     (dict(lists=64, n=0), -1), (dict(lists=64, n=4, tokens=2), -1), (dict(ws=None), -3), (dict(bytes=need - 1), -3),
                     (dict(ws=(1 << 22) + 4), -2), (dict(q=_vec(data=None)), -1), (dict(out=_vec(data=None)), -1), (dict(q=_vec(data=4)), -2),
                     (dict(out=_vec(head=4)), -2), (dict(q=_vec(token=12), tokens=2), -2), (dict(tokens=1 << 30), -6)):
        assert f(**kw) == code, kw
        if "lists" not in kw and "total" not in kw:
            assert f(**kw, prompt=True) == code, kw
    assert f(dtype=2, prompt=True) == -5 and f(scale=0.0, prompt=True) == -1 and f(scale=math.nan, prompt=True) == -1
    assert lib.leankv_byte_status(None, None) == -1


def test_select_checks_its_arguments():
    _no_gpu()
    lib = _native.byte_lib()

    def f(pool=None, q=None, dtype=0, **kw):
        a = {**dict(B=1, heads=8, ip=64, ids=64, pages=40, n=8, sinks=1, recent=2, blocks=64, out=64, scores=64, st=None), **kw}
        return lib.leankv_byte_select(ctypes.byref(pool or _pool()), dtype, ctypes.byref(q or _vec()), *a.values())

    for bad, code in BAD_POOLS:
        assert f(_pool(**bad)) == code
    for kw, code in ((dict(dtype=9), -1), (dict(B=0), -1), (dict(heads=3), -1), (dict(heads=64), -6), (dict(ip=None), -1), (dict(ids=None), -1),
                     (dict(pages=-1), -1), (dict(n=0), -1), (dict(sinks=-1), -1), (dict(recent=0), -1), (dict(sinks=7), -1), (dict(blocks=None), -1),
                     (dict(out=None), -1), (dict(scores=None), -1), (dict(B=1025), -6), (dict(q=_vec(data=None)), -1), (dict(q=_vec(data=8)), -2),
                     (dict(q=_vec(head=2)), -2)):
        assert f(**kw) == code, kw


def test_crop_checks_its_arguments():
    _no_gpu()
    lib = _native.lib()
    f = lambda **kw: lib.leankv_paged_table_crop(*{**dict(keep=1, B=1, n=64, table=64, pps=4, stack=64, top=64, size=4, status=64, st=None), **kw}.values())
    for kw, code in ((dict(keep=-1), -1), (dict(B=0), -1), (dict(B=1025), -6), (dict(pps=0), -1), (dict(size=0), -1), (dict(n=None), -1),
                     (dict(table=None), -1), (dict(stack=None), -1), (dict(top=None), -1), (dict(status=None), -1)):
        assert f(**kw) == code, kw
