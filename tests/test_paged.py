"""The paged serving operators' refusals (no GPU needed): bad arguments at the C entries before any launch, and the
Python checks."""
import pytest
import torch

EINVAL = 1


def _lib():
    import mimo_moe
    return mimo_moe.lib()


def test_header_is_bound():
    from test_cabi import declared_functions
    from mimo_moe._lib import SIGNATURES
    names = declared_functions("mimo_moe_paged.h")
    L = _lib()
    assert names and all(hasattr(L, n) and n in SIGNATURES for n in names)


A = 1 << 20   # an aligned address that no refused call touches


def plan_args(**kw):
    d = dict(lens=A, new=A + 64, R=2, table=A, width=4, free=A, n_free=A + 128, pages=8, P=16, T=4, cu=A, seq=A + 256,
             n_out=A + 512, pos=A, slots=A, status=None, stream=None)
    d.update(kw)
    return list(d.values())


@pytest.mark.parametrize("bad", [dict(lens=None), dict(new=None), dict(table=None), dict(free=None), dict(n_free=None),
                                 dict(cu=None), dict(seq=None), dict(n_out=None), dict(pos=None), dict(slots=None),
                                 dict(R=0), dict(R=4097), dict(width=0), dict(pages=0), dict(P=0), dict(P=8), dict(P=48),
                                 dict(P=256), dict(T=-1), dict(seq=A), dict(seq=A + 64), dict(n_out=A + 128),
                                 dict(pages=1 << 28), dict(width=1 << 28), dict(T=(1 << 30) + 1)])
def test_page_plan_refuses(bad):
    assert _lib().mimo_moe_page_plan(*plan_args(**bad)) == EINVAL


@pytest.mark.parametrize("bad", [dict(done=None), dict(lens=None), dict(table=None), dict(free=None), dict(n_free=None),
                                 dict(R=0), dict(R=4097), dict(width=0), dict(pages=0), dict(P=20)])
def test_page_release_refuses(bad):
    d = dict(done=A, R=2, lens=A, table=A, width=4, free=A, n_free=A, pages=8, P=16, status=None, stream=None)
    d.update(bad)
    assert _lib().mimo_moe_page_release(*d.values()) == EINVAL


@pytest.mark.parametrize("bad", [dict(qkv=None), dict(q=None), dict(k=None), dict(v=None), dict(pos=None),
                                 dict(slots=None), dict(T=0), dict(nq=0), dict(nkv=0), dict(d=12), dict(dv=12),
                                 dict(rot=3), dict(rot=-2), dict(rot=194), dict(d=512, rot=258), dict(theta=0.0),
                                 dict(vs=-1.0), dict(vs=float("nan")), dict(pages=0), dict(P=100), dict(qkv=A + 8),
                                 dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(T=2**31 - 1),
                                 dict(nq=2**31 - 1), dict(nq=1 << 26, nkv=1 << 26), dict(nkv=1 << 23)])
def test_paged_rope_store_refuses(bad):
    d = dict(qkv=A, T=4, nq=8, nkv=2, d=192, dv=128, rot=64, theta=1e4, vs=0.0, pos=A, slots=A, pages=8, P=16, q=A,
             k=A, v=A, status=None, stream=None)
    d.update(bad)
    assert _lib().mimo_moe_paged_rope_store(*d.values()) == EINVAL


@pytest.mark.parametrize("bad", [dict(cu=None), dict(seq=None), dict(plan=None), dict(R=0), dict(R=4097), dict(T=0),
                                 dict(nq=0), dict(nkv=0), dict(nkv=3), dict(nq=258, nkv=2), dict(window=-1),
                                 dict(keep=-1), dict(window=0, keep=4), dict(width=0), dict(P=8), dict(width=1 << 28),
                                 dict(plan=A + 8), dict(nb=-1), dict(T=(1 << 30) + 1)])
def test_paged_attention_plan_refuses(bad):
    L = _lib()
    d = dict(cu=A, seq=A, R=2, T=40, nq=8, nkv=2, window=128, keep=4, width=8, P=16, plan=A, nb=0, status=None,
             stream=None)
    d["nb"] = L.mimo_moe_paged_attention_plan_bytes(40, 2, 8, 2)
    assert d["nb"] > 0
    if bad.get("nb"):
        bad = dict(nb=d["nb"] - 1)
    d.update(bad)
    assert L.mimo_moe_paged_attention_plan(*d.values()) == EINVAL


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(plan=None),
                                 dict(out=None), dict(ws=None), dict(R=0), dict(R=4097), dict(T=0), dict(nkv=3),
                                 dict(nq=258, nkv=2), dict(d=96), dict(dv=192), dict(d=64), dict(scale=0.0),
                                 dict(scale=float("nan")), dict(window=-1), dict(keep=-1), dict(window=0, keep=4),
                                 dict(pages=0), dict(P=24), dict(width=0), dict(q=A + 8), dict(k=A + 2), dict(v=A + 8),
                                 dict(out=A + 16), dict(plan=A + 4), dict(ws=A + 16), dict(nb=-1), dict(wb=-1),
                                 dict(pages=1 << 26, nq=256, nkv=128, T=1), dict(T=2**31 - 1)])
def test_paged_attention_refuses(bad):
    L = _lib()
    d = dict(q=A, k=A, v=A, sinks=None, table=A, width=8, R=2, T=40, nq=8, nkv=2, d=192, dv=128, scale=0.1, window=128,
             keep=4, pages=8, P=16, plan=A, nb=0, out=A, ws=A, wb=0, status=None, stream=None)
    d.update({k: v for k, v in bad.items() if k not in ("nb", "wb")})
    d["nb"] = max(0, L.mimo_moe_paged_attention_plan_bytes(40, 2, 8, 2)) + 10**9 - 10**9 * (("nb" in bad) or 0)
    d["wb"] = 10**10 if "wb" not in bad else L.mimo_moe_paged_attention_workspace_bytes(40, 2, 8, 2, 128) - 1
    if "nb" in bad:
        d["nb"] -= 1
    assert L.mimo_moe_paged_attention(*d.values()) == EINVAL


def test_python_checks_refuse():
    from mimo_moe import paged
    from mimo_moe.layer import AttentionConfig
    cpu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.PageStep(block_table=torch.zeros(2, 4, dtype=torch.int32), page_size=16, cu_q=cpu, seq_lens=cpu,
                       positions=cpu, slots=cpu)
    with pytest.raises(ValueError):
        paged.page_plan(cpu, cpu, torch.zeros(2, 4, dtype=torch.int32), cpu, cpu[:1], 16, 4)
    with pytest.raises(ValueError):
        paged.page_release(torch.zeros(2, dtype=torch.bool), cpu, torch.zeros(2, 4, dtype=torch.int32), cpu, cpu[:1], 16)
    for kw in (dict(page_size=24), dict(max_requests=0), dict(max_requests=5000), dict(max_len=0), dict(num_pages=0),
               dict(num_pages=1 << 28)):
        with pytest.raises(ValueError):
            paged.PageTable(**{**dict(max_requests=4, max_len=64, num_pages=8, page_size=16, device="cpu"), **kw})
    with pytest.raises(ValueError):
        paged.PagedKVCache(AttentionConfig(), 4, 16, "cpu")
    with pytest.raises(ValueError):
        paged.PagedDecoderStack([], 4, 64, 8)


def test_ring_attention_refuses_first_tokens_that_stay():
    from mimo_moe.layer import AttentionConfig, KVCache, attention
    cfg = AttentionConfig(window=128, keep_first=4)
    with pytest.raises(ValueError):
        attention(torch.zeros(1, 64, 192), KVCache(cfg, 128, "cpu"), cfg, 0)


@pytest.mark.parametrize("bad", [dict(clear=A + 8), dict(width=0), dict(width=-8), dict(width=12), dict(width=(1 << 30) + 8),
                                 dict(q=None), dict(clear=A, T=0)])
def test_paged_rope_store_clear_refuses(bad):
    d = dict(qkv=A, T=4, nq=8, nkv=2, d=192, dv=128, rot=64, theta=1e4, vs=0.0, pos=A, slots=A, pages=8, P=16, q=A,
             k=A, v=A, clear=A, width=1024, status=None, stream=None)
    d.update(bad)
    assert _lib().mimo_moe_paged_rope_store_clear(*d.values()) == EINVAL


def test_first_tokens_that_stay_are_refused_before_a_ring_cache_is_touched():
    """By the cache itself, and by a layer given one that was made for another config, before it appends."""
    from mimo_moe.layer import Attention, AttentionConfig, DecoderLayer, DecoderStack, KVCache
    plain = AttentionConfig(n_heads=2, n_kv_heads=1, head_dim=64, v_head_dim=64, rotary_dim=32, window=128)
    cfg = AttentionConfig(n_heads=2, n_kv_heads=1, head_dim=64, v_head_dim=64, rotary_dim=32, window=128, keep_first=4)
    w = torch.zeros(128, 256, dtype=torch.bfloat16)
    attn = Attention(cfg, w, w[:64], w[:64], w.t())
    for make in (lambda: KVCache(cfg, 256, "cpu"), lambda: KVCache.for_layer(cfg, 256, device="cpu"),
                 lambda: DecoderLayer(attn, None, None, None).new_cache(256),
                 lambda: DecoderStack([DecoderLayer(attn, None, None, None)], 256)):
        with pytest.raises(ValueError, match="keep_first"):
            make()
    ring = KVCache(plain, 256, "cpu")
    with pytest.raises(ValueError, match="keep_first"):
        attn(torch.zeros(1, 256, dtype=torch.bfloat16), ring)
    assert ring.offset == 0 and not ring.k.any()


def test_a_cache_of_the_callers_own_needs_no_new_attribute():
    """A layer takes any object with a ring cache's members, as before there were paged ones."""
    from types import SimpleNamespace
    from mimo_moe.layer import Attention, AttentionConfig
    cfg = AttentionConfig(n_heads=2, n_kv_heads=1, head_dim=64, v_head_dim=64, rotary_dim=32)
    w = torch.zeros(128, 256, dtype=torch.bfloat16)
    attn = Attention(cfg, w, w[:64], w[:64], w.t())
    with pytest.raises(ValueError, match="cache slots"):   # the check of the ring's room: past the cache's kind
        attn(torch.zeros(5, 256, dtype=torch.bfloat16), SimpleNamespace(offset=0, cap=4))


def test_bf16_value_goes_by_the_value_alone():
    import math
    from mimo_moe.layer import bf16_value
    scale = torch.tensor(0.5)
    assert bf16_value(scale) == 0.5
    scale.fill_(0.707)
    assert bf16_value(scale) == bf16_value(0.707) == float(torch.tensor(0.707).to(torch.bfloat16))
    assert math.copysign(1, bf16_value(0.0)) == 1 and math.copysign(1, bf16_value(-0.0)) == -1
    assert math.isnan(bf16_value(math.nan)) and bf16_value(1e39) == math.inf and bf16_value(3) == 3.0


def test_a_step_that_does_not_fit_is_reported_in_its_own_words():
    from mimo_moe import paged, read_status
    from mimo_moe._lib import MIMO_ERANGE, MimoError
    step, stack = object.__new__(paged.PageStep), object.__new__(paged.PagedDecoderStack)
    stack.table = object.__new__(paged.PageTable)
    for holder, check in ((step, step.check), (stack.table, stack.check)):
        holder.status = torch.tensor([MIMO_ERANGE], dtype=torch.int32)
        with pytest.raises(ValueError, match="page") as e:
            check()
        assert "expert" not in str(e.value)
        check()                                   # cleared
        holder.status[0] = 5
        with pytest.raises(MimoError):
            check()
        check()
    with pytest.raises(ValueError, match="expert id"):   # a route's error keeps its words
        read_status(torch.tensor([MIMO_ERANGE], dtype=torch.int32), "router")


@pytest.mark.parametrize("T,R,nq,nkv", [(1 << 30, 1, 4096, 4096), (1 << 20, 1, 1 << 20, 1 << 20), (1 << 30, 4096, 2048, 128),
                                        (4096, 4096, 1 << 30, 1 << 30), (1 << 30, 1, 2**31 - 1, 2**31 - 1)])
def test_more_work_units_than_32_bits_number_are_refused(T, R, nq, nkv):
    """Their plan would be written past the bytes that were asked for."""
    L = _lib()
    assert L.mimo_moe_paged_attention_plan_bytes(T, R, nq, nkv) == 0
    assert L.mimo_moe_paged_attention_workspace_bytes(T, R, nq, nkv, 128) == 0
    assert L.mimo_moe_paged_attention_plan(A, A, R, T, nq, nkv, 0, 0, 8, 16, A, 1 << 60, None, None) == EINVAL
    assert L.mimo_moe_paged_attention(A, A, A, None, A, 8, R, T, nq, nkv, 192, 128, 0.1, 0, 0, 1, 16, A, 1 << 60, A, A,
                                      1 << 60, None, None) == EINVAL


def test_plan_bytes_grow_with_the_units():
    L = _lib()
    for T, R, nq, nkv in ((1 << 30, 1, 64, 4), (1 << 30, 4096, 128, 1), (1 << 20, 4096, 1024, 1024), (4096, 4096, 4096, 4096)):
        tok = 32 // (nq // nkv) if T <= R else 2 * (128 // (nq // nkv))
        assert L.mimo_moe_paged_attention_plan_bytes(T, R, nq, nkv) >= 32 * nkv * (T // tok)


def test_a_refused_layer_call_leaves_no_buffer_behind():
    """A cache that does not go with the step (another device, other pages) is refused before the step's scratch is made:
    a buffer of it, on the cache's device, would be what the next layer is given."""
    from mimo_moe import paged
    from mimo_moe.layer import AttentionConfig
    step = object.__new__(paged.PageStep)
    step.rows, step.tokens, step.page_size, step.device = paged._Rows(), 4, 16, torch.device("cuda", 0)
    cache = object.__new__(paged.PagedKVCache)
    cache.cfg, cache.page_size, cache.num_pages, cache.device = AttentionConfig(), 16, 8, torch.device("cpu")
    cache.step, cache.plan = step, None
    with pytest.raises(ValueError, match="pages of 16 on cpu"):
        cache.attend(torch.zeros(4, cache.cfg.qkv_width), None)
    assert not step.rows._bufs
