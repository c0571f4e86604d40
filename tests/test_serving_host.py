"""Refusals of the serving operators, without a GPU: arguments are checked before anything is launched."""
import ctypes

import pytest
import torch

from conftest import pkg

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def ops(monkeypatch):
    """The operators with CPU tensors let through the device check: what passes the checks ends at the library's own."""
    pkg("build").build()
    m = pkg("operators")
    monkeypatch.setattr(m, "_on_current_device", lambda *t: None)
    monkeypatch.setattr(m, "_stream", lambda: 0)
    return m


def cache(pages=4, Hk=2, page=16, D=64, B=2, width=2, dtype=BF16):
    return dict(k_pages=torch.zeros(pages, Hk, page, D, dtype=dtype), v_pages=torch.zeros(pages, Hk, page, D, dtype=dtype),
                page_table=torch.zeros(B, width, dtype=I32), lengths=torch.zeros(B, dtype=I32))


def rows(H=2, B=2, T=1, D=64, dtype=BF16):
    return torch.zeros(B, H, T, D, dtype=dtype)


def test_cpu_tensors_are_refused():
    m = pkg("operators")
    c = cache()
    for call in (lambda: m.attn_decode(rows(), **c), lambda: m.kv_append(rows(), rows(), **c),
                 lambda: m.kv_evict(*c.values(), torch.zeros(2, 2, 32), 8),
                 lambda: m.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=I32), torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_another_device_is_refused(monkeypatch):
    m = pkg("operators")

    class Elsewhere:
        is_cuda = True
        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    with pytest.raises(RuntimeError, match="cuda:1, but cuda:0"):
        m._on_current_device(None, Elsewhere())


def test_good_arguments_reach_the_device_check(ops):
    if torch.cuda.is_available():
        pytest.skip("host addresses must not reach a GPU")
    c = cache()
    w = torch.zeros(2, 2, 32)
    for call in (lambda: ops.attn_decode(rows(4), **c, k=rows(), v=rows(), weights=w), lambda: ops.kv_append(rows(), rows(), **c),
                 lambda: ops.kv_evict(*c.values(), w, 8),
                 lambda: ops.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=I32), torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match="sm_100"):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(k_pages=torch.zeros(4, 2, 16, 64)), TypeError),
    (dict(k_pages=torch.zeros(4, 2, 16, 64, dtype=torch.float16), v_pages=torch.zeros(4, 2, 16, 64, dtype=torch.float16)), TypeError),
    (dict(k_pages=torch.zeros(4, 2, 8, 64, dtype=BF16)), ValueError),
    (dict(k_pages=torch.zeros(4, 16, 64, dtype=BF16), v_pages=torch.zeros(4, 16, 64, dtype=BF16)), ValueError),
    (dict(v_pages=torch.zeros(4, 2, 64, 16, dtype=BF16).transpose(2, 3)), ValueError),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(2, 4, dtype=I32)[:, ::2]), ValueError),
    (dict(page_table=torch.zeros(1, 2, dtype=I32).expand(2, 2)), RuntimeError),
    (dict(page_table=torch.zeros(2, 0, dtype=I32)), RuntimeError),
    (dict(lengths=torch.zeros(3, dtype=I32)), ValueError),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(lengths=torch.zeros(4, dtype=I32)[::2]), ValueError),
    (dict(q=rows(3)), ValueError),
    (dict(q=rows(D=32)), ValueError),
    (dict(q=rows(B=3)), ValueError),
    (dict(q=rows(dtype=F32)), TypeError),
    (dict(q=rows(D=128)[..., ::2]), ValueError),
    (dict(k=rows()), RuntimeError),
    (dict(k=rows(3), v=rows(3)), ValueError),
    (dict(k=rows(T=2), v=rows(T=2)), ValueError),
    (dict(counts=torch.zeros(3, dtype=I32)), ValueError),
    (dict(counts=torch.zeros(2)), ValueError),
    (dict(counts=torch.zeros(4, dtype=I32)[::2]), ValueError),
    (dict(weights=torch.zeros(2, 2, 31)), ValueError),
    (dict(weights=torch.zeros(2, 2, 32, dtype=BF16)), ValueError),
    (dict(weights=torch.zeros(2, 3, 32)), ValueError),
    (dict(weights=torch.zeros(2, 2, 64)[:, :, ::2]), ValueError),
    (dict(weights=torch.zeros(2, 2, 32), weights_out=torch.zeros(2, 2, 33)), ValueError),
    (dict(p=1.5), RuntimeError),
    (dict(p=float("nan")), RuntimeError),
    (dict(out=rows(dtype=F32)), TypeError),
    (dict(out=rows(4)), ValueError),
])
def test_attention_refusals(ops, change, error):
    before = pkg("_lib").launch_count()
    args = dict(q=rows(), **cache())
    args.update(change)
    with pytest.raises(error):
        ops.attn_decode(**args)
    assert pkg("_lib").launch_count() == before


def test_head_size_limit(ops):
    with pytest.raises(RuntimeError, match="bad shape"):
        ops.attn_decode(rows(D=264), **cache(D=264))


def test_empty_batches_return_empty(ops):
    c = cache(B=0)
    assert ops.attn_decode(rows(B=0), **c).shape == (0, 2, 1, 64)
    assert ops.attn_decode(rows(T=0), **cache()).shape == (2, 2, 0, 64)
    ops.kv_append(rows(B=0), rows(B=0), **c)
    kept, new = ops.kv_evict(*c.values(), torch.zeros(0, 2, 32), 8)
    assert kept.shape == (0, 2, 8) and new.shape == (0,)
    tokens, n = ops.verify_drafts(torch.zeros(0, 3, 8), torch.zeros(0, 2, dtype=I32), torch.zeros(0, 3))
    assert tokens.shape == (0, 3) and n.shape == (0,)


@pytest.mark.parametrize("change,error", [
    (dict(budget=0), ValueError), (dict(recent=-1), ValueError), (dict(recent=9), ValueError),
    (dict(weights=torch.zeros(2, 2, 31)), ValueError), (dict(weights=torch.zeros(2, 2, 32, dtype=torch.float64)), ValueError),
    (dict(weights_out=torch.zeros(2, 2, 7)), ValueError), (dict(dst_table=torch.zeros(2, 0, dtype=I32)), ValueError),
    (dict(dst_table=torch.zeros(1, 2, dtype=I32)), ValueError), (dict(dst_table=torch.zeros(2, 2)), ValueError),
    (dict(dst_table=torch.zeros(1, 1, dtype=I32).expand(2, 1)), RuntimeError),
])
def test_eviction_refusals(ops, change, error):
    args = dict(**cache(), weights=torch.zeros(2, 2, 32), budget=8, recent=2)
    args.update(change)
    with pytest.raises(error):
        ops.kv_evict(**args)


@pytest.mark.parametrize("change,error", [
    (dict(target_probs=torch.zeros(2, 8)), ValueError), (dict(target_probs=torch.zeros(2, 3, 8, dtype=torch.float64)), (TypeError, ValueError)),
    (dict(target_probs=torch.zeros(2, 8, 3).transpose(1, 2)), ValueError), (dict(target_probs=torch.zeros(2, 4, 8)), ValueError),
    (dict(draft_tokens=torch.zeros(2, 2, dtype=torch.int64)), ValueError), (dict(uniforms=torch.zeros(2, 2)), ValueError),
    (dict(uniforms=torch.zeros(2, 3, dtype=torch.float64)), ValueError), (dict(draft_probs=torch.zeros(2, 3, 8)), ValueError),
    (dict(draft_probs=torch.zeros(2, 2, 8, dtype=BF16)), ValueError), (dict(counts=torch.zeros(2)), ValueError),
    (dict(counts=torch.zeros(3, dtype=I32)), ValueError),
])
def test_verification_refusals(ops, change, error):
    args = dict(target_probs=torch.zeros(2, 3, 8), draft_tokens=torch.zeros(2, 2, dtype=I32), uniforms=torch.zeros(2, 3))
    args.update(change)
    with pytest.raises(error):
        ops.verify_drafts(**args)


def test_library_refuses_on_its_own():
    """The C entry points check what a caller without the Python layer may get wrong; nothing is launched."""
    pkg("build").build()
    m = pkg("_lib")
    lib = m.lib()
    before = lib.ptj_launch_count()
    good = lambda **kw: m.KvCache(**{**dict(k=16, v=16, table=16, lengths=16, batch=2, kv_heads=2, d_head=64, pages=4, page_size=16,
                                            table_width=2, table_ld=2, k_strides=(2048, 1024, 64), v_strides=(2048, 1024, 64),
                                            dtype=m.PTJ_BF16), **kw})
    new = lambda **kw: m.NewTokens(**{**dict(q=16, k=None, v=None, out=16, counts=None, heads=4, tokens=1, q_strides=(256, 64, 64),
                                             o_strides=(256, 64, 64), k_strides=(0, 0, 0), v_strides=(0, 0, 0)), **kw})
    call = lambda c, t, p=0.1, w=None, wo=None, ld=0: lib.ptj_attn_decode(
        ctypes.byref(c) if c else None, ctypes.byref(t) if t else None, p, w, wo, ld, None, 0, None)
    assert call(None, new()) == -1 and call(good(), None) == -1
    for kw in (dict(k=None), dict(table=None), dict(lengths=None), dict(batch=0), dict(batch=-1), dict(kv_heads=0), dict(d_head=0),
               dict(d_head=257), dict(pages=0), dict(page_size=0), dict(table_width=0), dict(table_ld=1), dict(k_strides=(-1, 0, 0)),
               dict(table_width=1 << 28, table_ld=1 << 28)):
        assert call(good(**kw), new()) == -1, kw
    assert call(good(dtype=7), new()) == -3
    for kw in (dict(q=None), dict(out=None), dict(heads=3), dict(heads=0), dict(tokens=0), dict(k=16), dict(v=16), dict(tokens=5000),
               dict(q_strides=(0, -1, 0))):
        assert call(good(), new(**kw)) == -1, kw
    assert call(good(), new(), p=1.1) == -1 and call(good(), new(), w=16, wo=None) == -1
    assert call(good(), new(), wo=16, ld=31) == -1
    long = dict(table_width=4096, table_ld=4096, batch=1, kv_heads=1)
    need = lib.ptj_attn_decode_workspace_bytes(ctypes.byref(good(**long)), ctypes.byref(new(heads=1)), 0)
    assert need > 0 and call(good(**long), new(heads=1)) == -5
    assert lib.ptj_attn_decode(ctypes.byref(good(**long)), ctypes.byref(new(heads=1)), 0.1, None, None, 0, 16, need - 1, None) == -5
    assert lib.ptj_attn_decode(ctypes.byref(good(**long)), ctypes.byref(new(heads=1)), 0.1, None, None, 0, 24, need, None) == -2
    assert lib.ptj_attn_decode_workspace_bytes(None, None, 0) == 0
    assert call(good(kv_heads=1), new(heads=4097)) == -1  # query rows of a key head
    assert lib.ptj_kv_append(ctypes.byref(good()), ctypes.byref(new()), None) == -1
    for o in ((0, 64, 64), (256, 0, 64)):  # sequences, heads that share their output
        assert call(good(), new(o_strides=o)) == -1
    shared = good(k_strides=(2048, 0, 64))  # heads that share their keys: read, not written
    assert call(shared, new(k=16, v=16)) == -1 and lib.ptj_kv_append(ctypes.byref(shared), ctypes.byref(new(k=16, v=16)), None) == -1
    assert lib.ptj_kv_evict(ctypes.byref(shared), 48, 1, 1, 8, 0, 16, 32, 16, 32, 16, 32, None) == -1
    evict = lambda dst=16, width=1, ld=2, budget=8, recent=0, w=16, wld=32, wo=16, wold=32, kept=16, nl=32: lib.ptj_kv_evict(
        ctypes.byref(good()), dst, width, ld, budget, recent, w, wld, wo, wold, kept, nl, None)
    for kw in (dict(dst=None), dict(width=0), dict(ld=0), dict(budget=0), dict(recent=9), dict(recent=-1), dict(w=None), dict(wld=31),
               dict(wold=7, wo=48), dict(wold=31), dict(kept=None), dict(nl=None), dict(nl=16), dict(budget=17),
               dict(ld=1)):  # (in place with rows of another length)
        assert evict(**kw) == -1, kw
    two = (ctypes.c_int64 * 2)(24, 8)
    verify = lambda t=16, ts=two, d=None, ds=None, tok=16, u=16, out=16, acc=16, B=2, K=2, V=8, dt=0: lib.ptj_verify_drafts(
        t, ctypes.byref(ts) if ts else None, d, ds, tok, None, u, out, acc, B, K, V, dt, None)
    for kw in (dict(t=None), dict(ts=None), dict(d=16), dict(tok=None), dict(u=None), dict(out=None), dict(acc=None), dict(B=0), dict(K=-1),
               dict(V=0)):
        assert verify(**kw) == -1, kw
    assert verify(dt=9) == -3
    assert lib.ptj_launch_count() == before


def test_cache_and_speculation_refusals():
    """What serving refuses before it touches a device."""
    sv, gpt2 = pkg("serving"), pkg("gpt2")
    cfg = gpt2.GPT2Config(vocab=10, dim=8, layers=1, heads=2, ffn=16, seq=32)
    for kw in (dict(batch=0), dict(batch=1, capacity=0), dict(batch=1, page_size=0)):
        with pytest.raises(ValueError):
            sv.PagedCache(cfg, device="cpu", **kw)
    c = sv.PagedCache(cfg, 2, capacity=20, page_size=16, device="cpu")
    assert tuple(c.page_table.shape) == (2, 2) and c.k.shape == (1, 4, 2, 16, 4)
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(4, 2)
    with pytest.raises(ValueError, match="sequences for a cache"):
        sv.decode_step((cfg, None), torch.zeros(3, 1, dtype=I32), c)
    with pytest.raises(ValueError, match="another model"):
        sv.decode_step((gpt2.GPT2Config(vocab=10, dim=16, layers=1, heads=2, ffn=16, seq=32), None), torch.zeros(2, 1, dtype=I32), c)


@pytest.mark.parametrize("change", [dict(drafts=0), dict(uniforms=torch.zeros(4, 2, 4)), dict(uniforms=torch.zeros(4, 3, 10)),
                                    dict(new_tokens=40), dict(budget=3, recent=4), dict(budget=0)])
def test_speculation_refusals(change, monkeypatch):
    sv, gpt2 = pkg("serving"), pkg("gpt2")
    cfg = gpt2.GPT2Config(vocab=10, dim=8, layers=1, heads=2, ffn=16, seq=32)
    monkeypatch.setattr(sv, "_weights", lambda params, dtype, p=None: (cfg, None))
    args = dict(params=[[torch.zeros(1)]], draft_params=[[torch.zeros(1)]], prompt=torch.zeros(2, 5, dtype=I32), new_tokens=8,
                uniforms=torch.zeros(4, 2, 10), drafts=4)
    args.update(change)
    with pytest.raises(ValueError):
        sv.speculate(**args)
