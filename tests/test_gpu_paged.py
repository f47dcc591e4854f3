"""The paged serving operators on the GPU (mimo_moe.paged) against plain 64-bit forms (tests/paged_ref.py).

Tolerances, element by element, with u = 2^-8 (half a bf16 step, relative):
  RoPE       u |ref| for the rounding of the result, plus 2^-22 (|x1| + |x2|): the float32 cosine, sine, products and
             sum before it (2^-24 each, less than four of them)
  attention  u |ref| for the result; (u + 2^-11) A with A = sum p |v| / sum p for the probabilities: u where they are
             rounded to bf16 for the product with V, 2^-11 for the float32 scores (a dot product of 192 values of
             about 1 is off by less than 192 * 2^-24 * sum |q k| scale ~ 1e-4) and the 2^x unit (2^-22)
"""
import numpy as np
import pytest
import torch

import paged_ref as PR

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
FULL = dict(n_heads=64, n_kv_heads=4, head_dim=192, v_head_dim=128, rotary_dim=64)
SWA = dict(n_heads=64, n_kv_heads=8, head_dim=192, v_head_dim=128, rotary_dim=64, rope_theta=10_000.0, window=128,
           sinks=True)
D128 = dict(n_heads=64, n_kv_heads=8, head_dim=128, v_head_dim=128, rotary_dim=128)
D64 = dict(n_heads=8, n_kv_heads=8, head_dim=64, v_head_dim=64, rotary_dim=32)
G3 = dict(n_heads=12, n_kv_heads=4, head_dim=128, v_head_dim=128, rotary_dim=128)        # 128 is no multiple of G
G128 = dict(n_heads=128, n_kv_heads=1, head_dim=192, v_head_dim=128, rotary_dim=64)
MHA = dict(n_heads=4, n_kv_heads=4, head_dim=192, v_head_dim=128, rotary_dim=64)


def i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def cfg_of(d, **kw):
    from mimo_moe.layer import AttentionConfig
    return AttentionConfig(**{**d, **kw})


# ------------------------------------------------------------------------------------------------ plan and release
def start(lens, P, width, spare, seed):
    """A random page assignment of requests holding lens tokens: (table, free list, n_free, num_pages)."""
    rng = np.random.default_rng(seed)
    used = [-(-h // P) for h in lens]
    N = sum(used) + spare
    perm = rng.permutation(N).tolist()
    table, k = [], 0
    for n in used:
        table.append(perm[k:k + n] + [-1] * (width - n))
        k += n
    return table, perm[k:] + [0] * k, N - k, N


PLANS = [
    # lens, new, page, padding rows
    ([0], [1], 16, 0),
    ([5], [0], 16, 3),
    ([15], [1], 16, 0),
    ([16], [1], 16, 1),
    ([0, 0, 0], [0, 0, 0], 64, 5),
    ([0, 0, 0], [0, 0, 0], 64, 0),
    ([4096] * 8, [1] * 8, 64, 0),
    ([1, 63, 64, 65, 0, 127, 128], [1, 1, 1, 1, 64, 0, 129], 64, 7),
    ([100, 0, 31, 7], [28, 300, 0, 1], 128, 0),
    (list(range(0, 700, 7)), [(i * i) % 37 for i in range(100)], 32, 11),
    ([i % 50 for i in range(1023)], [(i * 7) % 5 for i in range(1023)], 16, 1),
    ([i % 97 for i in range(4096)], [1 + (i % 40) for i in range(4096)], 16, 13),
    ([0], [70001], 16, 2),
]


@pytest.mark.parametrize("lens,new,P,pad", PLANS, ids=[f"R{len(p[0])}-T{sum(p[1])}-P{p[2]}" for p in PLANS])
def test_page_plan_matches_the_token_by_token_form(gpu, lens, new, P, pad):
    from mimo_moe import paged
    width = max(-(-(h + n) // P) for h, n in zip(lens, new)) + 2
    need = sum(-(-(h + n) // P) - -(-h // P) for h, n in zip(lens, new))
    table, free, n_free, N = start(lens, P, width, need + 3, len(lens))
    T = sum(new) + pad
    want = PR.plan(lens, new, table, free, n_free, P, T)
    args = [i32(x, gpu) for x in (lens, new, table, free, [n_free])]
    for again in range(2):                    # lens and n_free are inputs: a second plan is the same plan
        step = paged.page_plan(args[0], args[1], args[2], args[3], args[4], P, T)
        got = (step.cu_q, step.seq_lens, step.n_free, step.positions, step.slots, args[2])
        for g, w, name in zip(got, want, ("cu_q", "seq_lens", "n_free", "positions", "slots", "table")):
            assert g.cpu().tolist() == (w if name != "n_free" else [w]), name
        step.check()
        assert args[0].tolist() == lens and args[4].tolist() == [n_free]
    assert step.last_rows().tolist() == [c - 1 for c in want[0][1:]]


def test_page_plan_takes_the_last_free_page_exactly(gpu):
    from mimo_moe import paged
    table, free, n_free, N = start([0, 0], 16, 4, 5, 1)
    t = i32(table, gpu)
    step = paged.page_plan(i32([0, 0], gpu), i32([48, 32], gpu), t, i32(free, gpu), i32([5], gpu), 16, 80)
    step.check()
    assert step.n_free.tolist() == [0] and sorted(t.flatten().tolist())[-5:] == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("lens,new,n_free,T,why", [
    ([0, 0], [48, 33], 5, 100, "one page short"),
    ([0, 0], [48, 32], 5, 79, "one row short"),
    ([0, 3], [-1, 2], 5, 10, "negative new length"),
    ([-2, 3], [1, 2], 5, 10, "negative length"),
    ([60, 3], [5, 2], 5, 10, "longer than the table row"),
    ([0, 0], [2**31 - 1, 2**31 - 1], 5, 10, "lengths whose sum passes 32 bits"),
    ([2**31 - 1, 0], [2**31 - 1, 1], 5, 10, "a length that passes 32 bits"),
    ([0, 0], [1, 1], 9, 10, "more free pages than the pool has"),
    ([0, 0], [1, 1], -1, 10, "a negative number of free pages"),
])
def test_page_plan_refuses_on_the_device_and_changes_nothing(gpu, lens, new, n_free, T, why):
    from mimo_moe import paged
    t = i32([[7, -1, -1, -1], [6, -1, -1, -1]], gpu)
    before = t.clone()
    step = paged.page_plan(i32(lens, gpu), i32(new, gpu), t, i32([0, 1, 2, 3, 4, 0, 0, 0], gpu), i32([n_free], gpu),
                           16, T)
    assert torch.equal(t, before)
    assert step.cu_q.tolist() == [0, 0, 0] and step.seq_lens.tolist() == lens and step.n_free.tolist() == [n_free]
    assert set(step.positions.tolist()) == {-1} and set(step.slots.tolist()) == {-1}
    with pytest.raises(ValueError):
        step.check()
    step.check()     # cleared


def test_page_plan_reports_a_page_outside_the_pool(gpu):
    from mimo_moe import paged
    t = i32([[9, -1], [1, -1]], gpu)          # request 0 sits in page 9 of a pool of 4
    step = paged.page_plan(i32([3, 3], gpu), i32([2, 2], gpu), t, i32([0, 2, 3, 0], gpu), i32([3], gpu), 16, 4)
    assert step.slots.tolist() == [-1, -1, 19, 20]
    with pytest.raises(ValueError):
        step.check()


def test_page_release_and_a_long_run_of_steps(gpu):
    """Requests come, grow and go for 60 steps: the table equals a host copy of the same rules, no page is held twice,
    and all pages are back at the end."""
    from mimo_moe import paged
    R, P, N, T = 37, 16, 400, 300
    table = paged.PageTable(R, 20 * P, N, P, gpu)
    rng = np.random.default_rng(3)
    lens, host, free = [0] * R, [[-1] * 20 for _ in range(R)], list(range(N - 1, -1, -1))
    for it in range(60):
        new = []
        for r in range(R):
            n = int(rng.integers(0, 30)) if lens[r] == 0 else int(rng.integers(0, 3))
            new.append(min(n, 20 * P - lens[r], T - sum(new)))
        step = table.step(i32(new, gpu), T)
        cu, lens, left, pos, slots, host = PR.plan(lens, new, host, free, len(free), P, T)
        free = free[:left]
        assert step.positions.tolist() == pos and step.slots.tolist() == slots, it
        done = [bool(rng.random() < 0.1) for _ in range(R)]
        table.release(torch.tensor(done, device=gpu))
        for r in range(R):
            if done[r]:
                free += [p for p in host[r] if p >= 0]
                host[r], lens[r] = [-1] * 20, 0
        assert table.block_table.tolist() == host and table.lens.tolist() == lens
        assert table.n_free.tolist() == [len(free)] and table.free_pages.tolist()[:len(free)] == free
        held = [p for row in host for p in row if p >= 0]
        assert len(set(held + free)) == N
    table.release(torch.ones(R, dtype=torch.uint8, device=gpu))
    assert table.n_free.tolist() == [N] and sorted(table.free_pages.tolist()) == list(range(N))
    step.check()


@pytest.mark.parametrize("lens,table,n_free,why", [
    ([65, 1], [[0, 1, 2, 3], [4, -1, -1, -1]], 3, "a length outside the table"),
    ([20, 1], [[0, 8, -1, -1], [4, -1, -1, -1]], 3, "a page outside the pool"),
    ([20, 1], [[0, -1, -1, -1], [4, -1, -1, -1]], 3, "a page that is not there"),
    ([20, 1], [[0, 1, -1, -1], [4, -1, -1, -1]], 6, "more pages than the pool has"),
])
def test_page_release_refuses_on_the_device_and_changes_nothing(gpu, lens, table, n_free, why):
    from mimo_moe import paged
    state = [i32(lens, gpu), i32(table, gpu), i32([7, 6, 5, 0, 0, 0, 0, 0], gpu), i32([n_free], gpu)]
    before = [t.clone() for t in state]
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    paged.page_release(torch.tensor([True, True], device=gpu), *state, 16, status)
    assert int(status) == 2 and all(torch.equal(a, b) for a, b in zip(state, before))


# ------------------------------------------------------------------------------------------------------ RoPE + append
def layout(held, new, P, gpu, seed, pad=0, spare=3):
    """A PageStep of requests holding `held` and bringing `new` tokens over shuffled pages, and its pool's size."""
    from mimo_moe import paged
    total = [h + n for h, n in zip(held, new)]
    width = max(1, max(-(-t // P) for t in total)) + 1
    table, free, n_free, N = start(total, P, width, spare, seed)
    cu = [0]
    pos, slots = [], []
    for r, (h, n) in enumerate(zip(held, new)):
        cu.append(cu[-1] + n)
        pos += range(h, h + n)
        slots += [table[r][p // P] * P + p % P for p in range(h, h + n)]
    step = paged.PageStep(block_table=i32(table, gpu), page_size=P, cu_q=i32(cu, gpu), seq_lens=i32(total, gpu),
                          positions=i32(pos + [-1] * pad, gpu), slots=i32(slots + [-1] * pad, gpu))
    return step, table, N


ROPES = [
    # dims, held, new, page, padding rows, value scale
    (FULL, [0], [1], 16, 0, None),
    (FULL, [4096] * 8, [1] * 8, 64, 0, 0.707),
    (SWA, [0, 17, 300], [5, 1, 30], 16, 3, 0.707),
    (FULL, [100], [300], 128, 1, None),
    (SWA, [1000, 0], [150, 421], 32, 0, 0.707),
    (D128, [7, 0, 0], [33, 0, 2], 64, 2, None),
    (D64, [700], [9], 16, 0, 0.5),
    (dict(SWA, rotary_dim=34), [3, 0], [12, 9], 16, 1, None),
    (dict(FULL, rotary_dim=100), [9], [20], 32, 0, None),
    (dict(FULL, rotary_dim=160), [2_000_000], [3], 64, 0, None),
    (dict(FULL, rotary_dim=0), [5], [4], 64, 0, None),
    (dict(n_heads=3, n_kv_heads=1, head_dim=40, v_head_dim=24, rotary_dim=8), [0, 4], [50, 1], 16, 5, 0.707),
    (MHA, [40], [2500], 16, 0, None),
    (FULL, [3, 0], [900, 500], 64, 300, 0.707),                           # several rows a CTA, the last ones padding
    (dict(FULL, n_heads=200), [0], [200], 16, 200, 0.5),                  # rows of 80 KB
    (dict(FULL, n_heads=560, n_kv_heads=2), [11], [150], 16, 1, 0.5),     # of 217 KB
    (dict(FULL, n_heads=600, n_kv_heads=4), [1], [150], 16, 1, 0.5),      # wider than shared memory
    (dict(D128, n_heads=1, n_kv_heads=1), [0], [5000], 128, 7, 0.5),
    (dict(n_heads=2, n_kv_heads=2, head_dim=256, v_head_dim=8, rotary_dim=256), [100], [300], 16, 1, None),
]


@pytest.mark.parametrize("dims,held,new,P,pad,vs", ROPES)
def test_rope_store_paged_matches_the_plain_form(gpu, dims, held, new, P, pad, vs):
    from mimo_moe import paged
    from mimo_moe.layer import bf16_value
    cfg = cfg_of(dims, v_scale=vs)
    if max(held) > 100_000:      # a far position: its pages before it need not exist
        from mimo_moe.paged import PageStep
        n = sum(new)
        step = PageStep(block_table=i32([[0]], gpu), page_size=P, cu_q=i32([0, n], gpu), seq_lens=i32([n], gpu),
                        positions=i32([held[0] + i for i in range(n)], gpu), slots=i32(list(range(n)), gpu))
        N = 2
    else:
        step, _, N = layout(held, new, P, gpu, 5, pad)
    n, T = sum(new), sum(new) + pad
    g = torch.Generator().manual_seed(n)
    qkv = torch.randn(T, cfg.qkv_width, generator=g).to(torch.bfloat16)
    qkv[n:] = float("nan")
    cache = paged.PagedKVCache(cfg, N, P, gpu)
    cache.k.fill_(7.0)
    cache.v.fill_(9.0)
    q0 = torch.full((T, cfg.n_heads, cfg.head_dim), 3.0, dtype=torch.bfloat16, device=gpu)
    q = paged.rope_store_paged(qkv.to(gpu), cfg, cache, step, q_out=q0)
    step.check()
    nq, nkv, d, dv = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, cfg.v_head_dim
    x, pos = PR.f64(qkv[:n]), PR.f64(step.positions[:n])
    ref, mag = PR.rope(x[:, :(nq + nkv) * d].reshape(n, nq + nkv, d), pos, cfg.rotary_dim, cfg.rope_theta)
    slots = step.slots[:n].long()
    got = np.concatenate([PR.f64(q[:n]), PR.f64(cache.k[slots // P, :, slots % P])], 1)
    assert (np.abs(got - ref) <= U * np.abs(ref) + 2.0 ** -22 * mag).all()
    # dims past the rotary ones and values: bit for bit
    assert np.array_equal(got[..., cfg.rotary_dim:], ref[..., cfg.rotary_dim:])
    v = qkv[:n, (nq + nkv) * d:].float().view(n, nkv, dv)
    if vs is not None:
        v = (v * bf16_value(vs)).to(torch.bfloat16).float()
    assert torch.equal(cache.v[slots // P, :, slots % P].float().cpu(), v)
    # padding rows and all other slots as they were
    assert (q[n:] == 3.0).all()
    rest = torch.ones(N * P, dtype=torch.bool, device=gpu)
    rest[slots] = False
    rest = rest.view(N, P)
    assert (cache.k.transpose(1, 2)[rest] == 7.0).all() and (cache.v.transpose(1, 2)[rest] == 9.0).all()


def test_rope_store_paged_equals_the_one_sequence_kernel(gpu):
    """Same rows, same positions: the bits of mimo_moe.layer.rope_store on >= 99.99% (both evaluate the rotation to
    better than float32), and never more than one bf16 step apart."""
    from mimo_moe import paged
    from mimo_moe.layer import KVCache, rope_store
    cfg = cfg_of(SWA, v_scale=0.707)
    T = 600
    qkv = torch.randn(T, cfg.qkv_width, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    step, table, N = layout([5000], [T], 16, gpu, 2)
    cache, ring = paged.PagedKVCache(cfg, N, 16, gpu), KVCache(cfg, 8192, gpu)
    q, q1 = paged.rope_store_paged(qkv, cfg, cache, step), rope_store(qkv, cfg, ring, 5000)
    s = step.slots.long()
    pairs = [(q, q1), (cache.k[s // 16, :, s % 16], ring.k[:, 5000:5600].transpose(0, 1)),
             (cache.v[s // 16, :, s % 16], ring.v[:, 5000:5600].transpose(0, 1))]
    for a, b in pairs:
        d = (a.contiguous().view(torch.int16).int() - b.contiguous().view(torch.int16).int()).abs()
        assert int(d.max()) <= 1 and float((d == 0).float().mean()) >= 0.9999


def test_rope_store_paged_reports_a_slot_outside_the_pool(gpu):
    from mimo_moe import paged
    cfg = cfg_of(D64)
    step, _, N = layout([0], [4], 16, gpu, 2, spare=0)
    step.slots[2] = N * 16 + 3
    cache = paged.PagedKVCache(cfg, N, 16, gpu)
    qkv = torch.ones(4, cfg.qkv_width, device=gpu, dtype=torch.bfloat16)
    q = paged.rope_store_paged(qkv, cfg, cache, step)
    assert torch.isfinite(q).all() and (cache.v != 0).any(-1).sum() == 3 * cfg.n_kv_heads
    with pytest.raises(ValueError):
        step.check()


# ----------------------------------------------------------------------------------------------------------- attention
def fill(cfg, held, new, P, gpu, seed, pad=0, poison=float("nan")):
    """A step, a cache whose unseen slots hold NaN (none of them belongs to the requests' positions), q and the plain
    inputs of each request."""
    from mimo_moe import paged
    step, table, N = layout(held, new, P, gpu, seed, pad)
    g = torch.Generator().manual_seed(seed)
    cache = paged.PagedKVCache(cfg, N, P, gpu)
    cache.k.fill_(poison)
    cache.v.fill_(poison)
    kv = []
    for r, (h, n) in enumerate(zip(held, new)):
        L = h + n
        K = torch.randn(L, cfg.n_kv_heads, cfg.head_dim, generator=g).to(torch.bfloat16)
        V = torch.randn(L, cfg.n_kv_heads, cfg.v_head_dim, generator=g).to(torch.bfloat16)
        p = torch.arange(L)
        page = torch.tensor(table[r])[p // P].to(gpu)
        cache.k[page, :, (p % P).to(gpu)] = K.to(gpu)
        cache.v[page, :, (p % P).to(gpu)] = V.to(gpu)
        kv.append((K, V))
    T = sum(new) + pad
    q = torch.randn(T, cfg.n_heads, cfg.head_dim, generator=g).to(torch.bfloat16)
    q[sum(new):] = float("nan")
    sinks = torch.randn(cfg.n_heads, generator=g) if cfg.sinks else None
    return step, cache, q, kv, sinks


def compare(cfg, out, q, kv, held, new, sinks, some=None, blocks=0):
    """blocks: of a row of more than a few thousand keys, whose float32 output is 8 accumulations a block, each off by
    at most a unit in the last place of the row's magnitude (rounded or cut off)."""
    row = 0
    for r, (h, n) in enumerate(zip(held, new)):
        if n and (some is None or r in some):
            K, V = kv[r]
            ref, mag = PR.attention(PR.f64(q[row:row + n]), PR.f64(K), PR.f64(V), h, cfg.scale, cfg.window,
                                    cfg.keep_first, None if sinks is None else PR.f64(sinks))
            got = PR.f64(out[row:row + n])
            bad = ~(np.abs(got - ref) <= U * np.abs(ref) + (U + 2.0 ** -11 + blocks * 2.0 ** -20) * mag)
            assert not bad.any(), (r, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.abs(got - ref).max()))
        row += n


ATTN = [
    # dims (+ window, keep_first), held, new, page, padding rows
    (FULL, [0], [1], 16, 0),
    (FULL, [15], [1], 16, 0),
    (FULL, [127], [1], 64, 0),
    (FULL, [128], [1], 64, 0),
    (FULL, [2000] * 8, [1] * 8, 64, 0),
    (FULL, [0, 5, 127, 128, 129, 1000, 3001], [1, 1, 1, 1, 1, 1, 1], 16, 2),
    (FULL, [3000, 0, 64, 900], [3, 0, 7, 1], 32, 0),
    (FULL, [0], [300], 64, 0),
    (FULL, [0], [16], 128, 1),
    (FULL, [250], [100], 16, 0),
    (FULL, [0, 700, 33], [40, 1, 129], 32, 5),
    (FULL, [4000], [37], 128, 0),
    (SWA, [0], [1], 16, 0),
    (SWA, [5000], [1], 16, 0),
    (SWA, [0, 100, 127, 128, 129, 500], [1, 1, 1, 1, 1, 1], 64, 0),
    (SWA, [0], [300], 16, 0),
    (SWA, [1000, 77], [200, 8], 32, 3),
    (dict(SWA, keep_first=4), [0, 3, 130, 131, 132, 133, 900], [1] * 7, 16, 0),
    (dict(SWA, keep_first=4), [0, 600], [400, 9], 64, 0),
    (dict(SWA, keep_first=200), [1000, 150, 310], [1, 200, 40], 16, 1),
    (dict(SWA, keep_first=100000), [700], [20], 32, 0),
    (dict(SWA, window=1), [0, 50], [5, 1], 16, 0),
    (dict(SWA, window=1, keep_first=1), [0, 50], [300, 1], 128, 0),
    (dict(SWA, window=1000, sinks=False), [2000, 0], [70, 1100], 64, 0),
    (D128, [90, 0], [40, 200], 64, 0),
    (D128, [1500, 3, 200], [1, 1, 1], 16, 4),
    (D64, [700, 0, 31], [5, 140, 1], 16, 0),
    (dict(D64, window=40, sinks=True, keep_first=3), [700, 0], [5, 260], 32, 2),
    (G3, [0, 400, 9], [100, 1, 43], 16, 0),
    (G128, [10, 700], [3, 1], 64, 0),
    (MHA, [100, 0, 1000], [300, 1, 1], 32, 0),
    (MHA, [0] * 5 + [200] * 20, [1] * 25, 16, 0),
    (dict(FULL, n_heads=8, n_kv_heads=1), [20000], [2], 16, 0),
    (dict(D64, n_heads=2, n_kv_heads=1), [i * 3 for i in range(300)], [1 + i % 3 for i in range(300)], 16, 9),
    # no more rows than requests, but all of one request's: several small units
    (FULL, [300] + [5] * 44, [37] + [0] * 44, 16, 0),
    (dict(SWA, keep_first=17), [700, 0] + [0] * 60, [29, 30] + [0] * 60, 32, 1),
    (dict(G3, window=50, sinks=True), [9, 1000, 0, 0], [1, 3, 0, 0], 128, 0),
    # windows of more blocks than a unit that is never cut has, and of as many
    (dict(SWA, window=1000, keep_first=200), [5000, 3000, 0], [1, 1, 700], 16, 0),
    (dict(G3, window=700), [4000, 300], [40, 1], 64, 2),
    (dict(D64, n_heads=1, n_kv_heads=1, window=257, keep_first=3, sinks=True), [4000, 90], [1, 1], 64, 0),
    # few rows over many keys: parts of every size
    (dict(FULL, n_heads=2, n_kv_heads=1), [30000, 200, 1], [1, 1, 1], 128, 0),
    (dict(D64, n_heads=1, n_kv_heads=1, sinks=True), [40000], [300], 64, 3),
]


@pytest.mark.parametrize("dims,held,new,P,pad", ATTN)
def test_attention_paged_matches_the_plain_form(gpu, dims, held, new, P, pad):
    from mimo_moe import paged
    cfg = cfg_of(dims)
    step, cache, q, kv, sinks = fill(cfg, held, new, P, gpu, 11 + len(held), pad)
    T = sum(new) + pad
    out = torch.full((T, cfg.n_heads, cfg.v_head_dim), 5.0, dtype=torch.bfloat16, device=gpu)
    got = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks, out=out)
    assert got is out
    step.check()
    compare(cfg, out, q, kv, held, new, sinks)
    assert (out[sum(new):] == 5.0).all()
    # without `out`, padding rows are zero; with a plan made beforehand, the same bits
    plan = paged.attention_plan(step, cfg)
    again = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks, plan=plan)
    assert torch.equal(again[:sum(new)], out[:sum(new)]) and (again[sum(new):] == 0).all()
    step.check()


def test_attention_paged_of_values_that_leave_the_softmax_narrow_or_flat(gpu):
    """Scores up to +-1000 (one key takes all), equal scores (a plain mean) and a sink that outweighs every key."""
    from mimo_moe import paged
    cfg = cfg_of(D128, sinks=True)
    held, new, P = [300, 0, 64], [9, 150, 1], 16
    step, cache, q, kv, sinks = fill(cfg, held, new, P, gpu, 4)
    sinks[:8], sinks[8:16], sinks[16:24] = 80.0, -80.0, -float("inf")
    q[:9] *= 100.0
    q[9:159] = 0.0
    out = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks)
    step.check()
    # scores of +-1000 are off by 192 * 2^-24 * 1000 * 1.6 ~ 0.02 before the exponential: compare those rows as means
    row = PR.attention(PR.f64(q[:9]), PR.f64(kv[0][0]), PR.f64(kv[0][1]), 300, cfg.scale, sinks=PR.f64(sinks))
    assert (np.abs(PR.f64(out[:9]) - row[0]) <= U * np.abs(row[0]) + (U + 0.05) * row[1]).all()
    compare(cfg, out, q, kv, held, new, sinks, some=(1, 2))


def test_attention_paged_does_not_read_what_no_query_sees(gpu):
    """Pages before a window may be gone (-1 entries, or another request's page full of NaN)."""
    from mimo_moe import paged
    cfg = cfg_of(SWA, keep_first=4)
    held, new, P = [1000, 700], [3, 40], 16
    step, cache, q, kv, sinks = fill(cfg, held, new, P, gpu, 8)
    want = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks)
    step.block_table[0, 1:(1000 - 127) // P] = -1
    step.block_table[1, 1:(700 - 127) // P] = 2**30
    got = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks)
    step.check()
    assert torch.equal(got, want)


def test_attention_paged_reports_what_does_not_fit_and_serves_the_rest(gpu):
    from mimo_moe import paged
    cfg = cfg_of(D128)
    held, new, P = [100, 50, 0], [2, 3, 20], 16
    step, cache, q, kv, _ = fill(cfg, held, new, P, gpu, 9)
    for name, at, value in (("seq_lens", 1, 2), ("seq_lens", 1, 100000), ("seq_lens", 1, -5)):
        was = int(getattr(step, name)[at])
        getattr(step, name)[at] = value
        out = paged.attention_paged(q.to(gpu), cache, cfg, step)
        with pytest.raises(ValueError):
            step.check()
        compare(cfg, out, q, kv, held, new, None, some=(0, 2))
        assert (out[2:5] == 0).all(), (name, value)
        getattr(step, name)[at] = was
    was = int(step.block_table[1, 0])
    for page in (-1, 10**6):
        step.block_table[1, 0] = page
        out = paged.attention_paged(q.to(gpu), cache, cfg, step)
        with pytest.raises(ValueError):
            step.check()
        compare(cfg, out, q, kv, held, new, None, some=(0, 2))
    step.block_table[1, 0] = was
    # row offsets that run past the rows, or backwards
    for cu in ([0, 2, 5, 4000], [0, 2, -7, 25], [0, 30, 5, 25], [-3, 2, 5, 25]):
        step.cu_q.copy_(i32(cu, gpu))
        out = paged.attention_paged(q.to(gpu), cache, cfg, step)
        with pytest.raises(ValueError):
            step.check()
        assert out.shape[0] == 25


def test_attention_paged_takes_other_layouts_streams_and_two_calls_at_once(gpu):
    from mimo_moe import paged
    cfg = cfg_of(FULL)
    held, new, P = [3000, 200, 1], [1, 150, 1], 16
    step, cache, q, kv, _ = fill(cfg, held, new, P, gpu, 21)
    want = paged.attention_paged(q.to(gpu), cache, cfg, step)
    wide = torch.zeros(q.shape[0], 2 * cfg.n_heads, cfg.head_dim, dtype=torch.float32, device=gpu)
    wide[:, ::2] = q.to(gpu).float()
    assert torch.equal(paged.attention_paged(wide[:, ::2], cache, cfg, step), want)
    step2, cache2, q2, kv2, _ = fill(cfg, [900, 33], [200, 1], 64, gpu, 22)
    want2 = paged.attention_paged(q2.to(gpu), cache2, cfg, step2)
    qa, qb = q.to(gpu), q2.to(gpu)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            outs.append((paged.attention_paged(qa, cache, cfg, step), want))
        with torch.cuda.stream(s2):
            outs.append((paged.attention_paged(qb, cache2, cfg, step2), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)


def test_attention_paged_in_two_graphs_replayed_in_turn(gpu):
    """Two captured graphs with larger eager calls between their replays: each keeps its results."""
    from mimo_moe import paged
    cfg = cfg_of(FULL)
    runs = []
    for seed, held, new in ((1, [2000, 17], [1, 1]), (2, [500], [333])):
        step, cache, q, kv, _ = fill(cfg, held, new, 32, gpu, seed)
        q = q.to(gpu)
        out = torch.zeros(q.shape[0], cfg.n_heads, cfg.v_head_dim, dtype=torch.bfloat16, device=gpu)
        want = paged.attention_paged(q, cache, cfg, step)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged.attention_paged(q, cache, cfg, step, out=out)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged.attention_paged(q, cache, cfg, step, out=out)
        runs.append((g, out, want, step, cache, q))
    big = fill(cfg, [4000], [900], 64, gpu, 3)
    for _ in range(3):
        for g, out, want, *_ in runs:
            out.zero_()
            g.replay()
            paged.attention_paged(big[2].to(gpu), big[1], cfg, big[0])
            assert torch.equal(out, want)


# -------------------------------------------------------------------------------------------- the operators together
def stack_layers(gpu, hidden=1024):
    from mimo_moe.layer import AttentionConfig, DecoderLayer, synthetic_attention, synthetic_dense_mlp
    cfgs = [AttentionConfig(n_heads=16, n_kv_heads=2, v_scale=0.707),
            AttentionConfig(n_heads=16, n_kv_heads=4, rope_theta=10_000.0, window=128, sinks=True, v_scale=0.707)]
    return [DecoderLayer(synthetic_attention(c, hidden, seed=80 + i, device=gpu),
                         synthetic_dense_mlp(hidden, 1024, seed=90 + i, device=gpu), None, None)
            for i, c in enumerate(cfgs)]


def test_paged_stack_serves_each_request_as_a_stack_of_its_own(gpu):
    """Prompts in chunks, decoding and finished requests mixed over 8 steps, against a DecoderStack per request (the
    same kernels' family on a ring cache): max |d| / max |ref| <= 1e-2, the bar of the layer tests; a graph captured
    for the decode step serves the following tokens."""
    from mimo_moe.layer import DecoderStack
    from mimo_moe.paged import PagedDecoderStack
    layers = stack_layers(gpu)
    R, T = 5, 200
    stack = PagedDecoderStack(layers, max_requests=R, max_len=512, num_pages=80, page_size=16)
    g = torch.Generator().manual_seed(5)
    alone = [DecoderStack(layers, 512, 256) for _ in range(R)]

    def feed(new, rows, run=None):
        x = torch.zeros(rows, 1024, dtype=torch.bfloat16)
        x[:sum(new)] = torch.randn(sum(new), 1024, generator=g).to(torch.bfloat16)
        x = x.to(gpu)
        y = (run or stack)(x, i32(new, gpu))
        at = 0
        for r, n in enumerate(new):
            if n:
                ref = alone[r](x[at:at + n]).float()
                d = (y[at:at + n].float() - ref).abs().max() / ref.abs().max()
                assert float(d) <= 1e-2, (r, n, float(d))
                at += n

    feed([150, 3, 0, 20, 0], T)
    feed([40, 1, 130, 1, 0], T)
    feed([1, 1, 1, 1, 1], 5)
    assert stack.offset.tolist() == [191, 5, 131, 22, 1]
    stack.release(torch.tensor([False, True, False, True, False], device=gpu))
    for r in (1, 3):
        alone[r].at(0)
    feed([1, 60, 1, 17, 1], T)
    # a captured decode step: the lengths advance on the device
    xin, one = torch.zeros(5, 1024, dtype=torch.bfloat16, device=gpu), torch.ones(5, dtype=torch.int32, device=gpu)
    feed([1, 1, 1, 1, 1], 5)                    # the eager step first (cuBLAS and the buffers of this row count)
    graph = torch.cuda.CUDAGraph()
    state = stack.table._state.clone()
    with torch.cuda.graph(graph):
        y = stack(xin, one)
    assert torch.equal(stack.table._state, state)   # capture runs nothing

    def replay(x, new):
        xin.copy_(x)
        one.copy_(new)
        graph.replay()
        return y

    for _ in range(3):
        feed([1, 1, 1, 1, 1], 5, replay)
    feed([1, 0, 1, 1, 0], 5, replay)
    assert stack.offset.tolist() == [191 + 6, 60 + 4, 131 + 6, 17 + 5, 1 + 5]
    assert stack.table.last_rows().tolist() == [0, 0, 1, 2, 2]   # of the step [1, 0, 1, 1, 0]
    # more rows than any step before: buffers grow, and the graph keeps its own
    feed([60, 70, 1, 90, 20], 2 * T + 50)
    feed([1, 1, 1, 1, 1], 5, replay)
    stack.check()
    # a step that does not fit runs without new tokens and says so
    before = stack.offset.tolist()
    stack(torch.zeros(5, 1024, dtype=torch.bfloat16, device=gpu), i32([600, 0, 0, 0, 0], gpu))
    with pytest.raises(ValueError):
        stack.check()
    assert stack.offset.tolist() == before
    feed([1, 1, 1, 1, 1], 5, replay)
    stack.check()
    # rows of another width and steps without rows leave the lengths alone
    before = stack.offset.tolist()
    for bad in (torch.zeros(5, 1016, device=gpu), torch.zeros(1024, device=gpu), torch.zeros(5, 1024)):
        with pytest.raises(ValueError):
            stack(bad, i32([1, 1, 1, 1, 1], gpu))
    assert stack(torch.zeros(0, 1024, device=gpu), i32([0] * 5, gpu)).shape == (0, 1024)
    stack.check()
    assert stack.offset.tolist() == before


def test_python_refusals(gpu):
    from mimo_moe import paged
    from mimo_moe.layer import AttentionConfig
    cfg = cfg_of(SWA, keep_first=4)
    step, cache, q, kv, sinks = fill(cfg, [100, 20], [3, 1], 16, gpu, 1)
    q = q.to(gpu)
    plan = paged.attention_plan(step, cfg)
    other, *_ = fill(cfg, [100, 20], [3, 1], 16, gpu, 2)
    small = paged.PagedKVCache(cfg_of(D64), 20, 16, gpu)
    big_pages = paged.PagedKVCache(cfg, 20, 32, gpu)
    out = torch.empty(4, cfg.n_heads, cfg.v_head_dim, dtype=torch.bfloat16, device=gpu)
    odd = torch.empty(4 * cfg.n_heads * cfg.v_head_dim + 8, dtype=torch.bfloat16, device=gpu)[8:].view(out.shape)

    def att(**kw):
        a = dict(q=q, cache=cache, cfg=cfg, step=step, sinks=sinks, plan=plan, out=out)
        a.update(kw)
        return paged.attention_paged(**a)

    att()
    for kw in (dict(q=q[:3]), dict(q=q.cpu()), dict(step=other), dict(cfg=cfg_of(SWA)), dict(cfg=cfg_of(FULL)),
               dict(cache=small), dict(cache=big_pages), dict(sinks=sinks[:5]), dict(out=out.float()),
               dict(out=out[:, ::2]), dict(out=odd), dict(cfg=cfg_of(SWA, window=0, keep_first=4), plan=None),
               dict(cfg=cfg_of(SWA, window=-1), plan=None)):
        with pytest.raises(ValueError):
            att(**kw)
    for bad in (AttentionConfig(n_heads=6, n_kv_heads=4), AttentionConfig(n_heads=256, n_kv_heads=1),
                cfg_of(SWA, keep_first=-1)):
        with pytest.raises(ValueError):
            paged.attention_plan(step, bad)
    qkv = torch.zeros(4, cfg.qkv_width, dtype=torch.bfloat16, device=gpu)
    for args in ((qkv[:3], cfg, cache, step), (qkv[:, 8:], cfg, cache, step), (qkv, cfg, small, step),
                 (qkv, cfg_of(SWA, rotary_dim=33), cache, step)):
        with pytest.raises(ValueError):
            paged.rope_store_paged(*args)
    table = paged.PageTable(2, 64, 8, 16, gpu)
    for new, tokens in ((i32([1], gpu), 4), (i32([1, 1], gpu).long(), 4), (torch.ones(2, dtype=torch.int32), 4),
                        (i32([1, 1], gpu), -1)):
        with pytest.raises(ValueError):
            table.step(new, tokens)
    with pytest.raises(ValueError):
        table.release(torch.ones(3, dtype=torch.bool, device=gpu))
    assert table.lens.tolist() == [0, 0] and table.n_free.tolist() == [8]
    # no rows at all
    empty = table.step(i32([0, 0], gpu), 0)
    c0 = paged.PagedKVCache(cfg, 8, 16, gpu)
    assert paged.rope_store_paged(qkv[:0], cfg, c0, empty).shape[0] == 0
    assert paged.attention_paged(q[:0], c0, cfg, empty, sinks).shape[0] == 0
    empty.check()


def test_pages_far_into_a_pool_of_more_than_32_bits(gpu):
    """The last pages of a pool of 2^32 values and more give the bits that the same pages of a small pool give."""
    from mimo_moe import paged
    cfg, P, near = cfg_of(FULL), 128, 12
    far = 2**32 // (cfg.n_kv_heads * P * cfg.v_head_dim) + near
    held, new = [200, 300, 0], [3, 150, 1]
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(sum(new), cfg.qkv_width, generator=g).to(torch.bfloat16).to(gpu)
    got = []
    for N in (near, far):
        table = torch.tensor([[N - 1, N - 4, -1, -1], [N - 2, N - 3, N - 5, N - 6], [N - 7, -1, -1, -1]],
                             dtype=torch.int32, device=gpu)
        k = torch.empty(N, cfg.n_kv_heads, P, cfg.head_dim, dtype=torch.bfloat16, device=gpu)
        v = torch.empty(N, cfg.n_kv_heads, P, cfg.v_head_dim, dtype=torch.bfloat16, device=gpu)
        gen = torch.Generator(gpu).manual_seed(6)
        for t in (k, v):
            t[N - near:].copy_(torch.randn(t[N - near:].shape, generator=gen, device=gpu))
        cache = paged.PagedKVCache(cfg, N, P, k=k, v=v)
        step = paged.page_plan(i32(held, gpu), i32(new, gpu), table, torch.arange(N, dtype=torch.int32, device=gpu),
                               i32([N - 10], gpu), P, sum(new))
        q = paged.rope_store_paged(qkv, cfg, cache, step)
        out = paged.attention_paged(q, cache, cfg, step)
        step.check()
        got.append([t.cpu() for t in (q, out, k[N - near:], v[N - near:], step.slots - (N - near) * P)])
        del cache, k, v, t
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_rows_far_into_a_step_of_more_than_32_bits(gpu):
    """A prompt whose projection, q and output rows pass 2^31 values: its last rows."""
    from mimo_moe import paged
    cfg, P, n = cfg_of(SWA, sinks=False), 64, 48
    T = 2**31 // (cfg.n_heads * cfg.v_head_dim) + 2 * n + 5
    gen = torch.Generator(gpu).manual_seed(7)
    qkv = torch.empty(T, cfg.qkv_width, dtype=torch.bfloat16, device=gpu)
    for i in range(0, T, 16384):
        qkv[i:i + 16384].copy_(torch.randn(min(16384, T - i), cfg.qkv_width, generator=gen, device=gpu))
    table = paged.PageTable(1, T, -(-T // P), P, gpu)
    cache = paged.PagedKVCache(cfg, table.num_pages, P, gpu)
    step = table.step(i32([T], gpu), T)
    q = paged.rope_store_paged(qkv, cfg, cache, step)
    out = paged.attention_paged(q, cache, cfg, step)
    step.check()
    # the same rows alone: the rotation's bits, and the formula of the attention over the window they see
    one = paged.PageStep(block_table=step.block_table, page_size=P, cu_q=i32([0, n], gpu), seq_lens=i32([T], gpu),
                         positions=step.positions[-n:].contiguous(), slots=step.slots[-n:].contiguous())
    k0 = cache.k.clone()
    assert torch.equal(q[-n:], paged.rope_store_paged(qkv[-n:], cfg, cache, one))
    assert torch.equal(k0, cache.k)
    p = torch.arange(T - n - cfg.window, T, device=gpu)
    page = step.block_table[0][p // P].long()
    K, V = cache.k[page, :, p % P].cpu(), cache.v[page, :, p % P].cpu()
    # (positions counted from the first of these keys: the rows see the same of them)
    compare(cfg, out[-n:], q[-n:].cpu(), [(K, V)], [cfg.window], [n], None)


def test_attention_paged_in_a_call_of_seconds(gpu):
    """Waits are bounded, and none of them is for a whole call: a prompt of whole blocks, one page for all of them, and
    behind it a request whose last block is ragged."""
    from mimo_moe import paged
    cfg, P, T = cfg_of(dict(D64, n_heads=1, n_kv_heads=1)), 128, 3 * 2**20
    gen = torch.Generator(gpu).manual_seed(8)
    cache = paged.PagedKVCache(cfg, 2, P, gpu)
    cache.k.copy_(torch.randn(cache.k.shape, generator=gen, device=gpu))
    cache.v.copy_(torch.randn(cache.v.shape, generator=gen, device=gpu))
    small = 100
    table = torch.zeros(2, T // P, dtype=torch.int32, device=gpu)
    table[1] = 1
    q = torch.randn(T + small, 1, cfg.head_dim, generator=gen, device=gpu).to(torch.bfloat16)
    rows = torch.zeros(T + small, dtype=torch.int32, device=gpu)
    step = paged.PageStep(block_table=table, page_size=P, cu_q=i32([0, T, T + small], gpu),
                          seq_lens=i32([T, small], gpu), positions=rows, slots=rows)
    out = paged.attention_paged(q, cache, cfg, step)
    step.check()
    K, V = cache.k[1].transpose(0, 1)[:small].cpu(), cache.v[1].transpose(0, 1)[:small].cpu()
    compare(cfg, out[T:], q[T:].cpu(), [(K, V)], [0], [small], None)
    # a row that ends with the k-th repetition of the page sees every key k times: the softmax of the page alone
    K, V = cache.k[0].transpose(0, 1).cpu(), cache.v[0].transpose(0, 1).cpu()
    for k in (1, 1000, T // P):
        compare(cfg, out[k * P - 1:k * P], q[k * P - 1:k * P].cpu(), [(K, V)], [P - 1], [1], None, blocks=k)


@pytest.mark.parametrize("number", [lambda n: n, lambda n: n + 1, lambda n: 2**31 - 1, lambda n: -1, lambda n: -2**31],
                         ids=["n", "n + 1", "largest", "-1", "smallest"])
@pytest.mark.parametrize("dims", [D128, dict(SWA, window=400, keep_first=40)], ids=["full", "window"])
def test_attention_paged_reads_a_page_outside_the_pool_as_zeros(gpu, dims, number):
    """Every page number that is none of the pool's, the first one behind it among them: an error, and zeros for k and v,
    in a decoding request, a prompt's chunk and a split unit."""
    from mimo_moe import paged
    cfg = cfg_of(dims)
    held, new, P = [900, 600, 70, 9000], [1, 200, 1, 1], 16
    step, cache, q, kv, sinks = fill(cfg, held, new, P, gpu, 12)
    paged.attention_paged(q.to(gpu), cache, cfg, step, sinks)
    step.check()
    for r, pages in ((0, (0, 41, 55)), (1, (2, 30, 49)), (3, (1, 550, 562))):
        for j in pages:
            step.block_table[r, j] = number(cache.num_pages)
            for t in kv[r]:
                t[j * P:(j + 1) * P] = 0.0
    out = paged.attention_paged(q.to(gpu), cache, cfg, step, sinks)
    with pytest.raises(ValueError):
        step.check()
    compare(cfg, out, q, kv, held, new, sinks)


def attend_steps(gpu, dims, R=6, P=16):
    """A cache, its table and a function that runs attend on a step of given new lengths (rows of NaN where said)."""
    from mimo_moe import paged
    cfg = cfg_of(dims)
    sinks = torch.zeros(cfg.n_heads, device=gpu) if cfg.sinks else None
    table = paged.PageTable(R, 512, 80, P, gpu)
    cache = paged.PagedKVCache(cfg, 80, P, gpu)

    def run(new, rows, nan=()):
        qkv = torch.randn(rows, cfg.qkv_width, device=gpu, generator=torch.Generator(gpu).manual_seed(rows))
        for r in nan:
            qkv[r] = float("nan")
        cache.step = table.step(i32(new, gpu), rows)
        return cache.attend(qkv, sinks)

    return run, table, cache, sinks


@pytest.mark.parametrize("dims", [FULL, dict(SWA, rotary_dim=34), D64], ids=["full", "window, odd rotary", "d64"])
def test_padding_rows_of_a_layer_are_zero_whatever_the_rows_held_before(gpu, dims):
    """A request's NaN stays its own: the next, shorter step has zeros in the rows that held it."""
    run, table, cache, _ = attend_steps(gpu, dims)
    out = run([100, 2, 2, 0, 0, 30], 140, nan=range(104, 140))
    assert torch.isnan(out[104:134]).any() and torch.isfinite(out[:104]).all() and (out[134:] == 0).all()
    out = run([1, 0, 1, 0, 0, 0], 140)
    assert torch.isfinite(out[:2]).all() and (out[:2] != 0).any() and (out[2:] == 0).all()
    out = run([0] * 6, 140)
    assert (out == 0).all()
    cache.step.check()


def test_padding_rows_are_zero_in_a_buffer_that_a_capture_made(gpu):
    """A buffer made while a graph is captured lies in memory that an earlier graph left full of NaN; an eager padded
    step uses it before the graph's first replay, another one after."""
    run, table, cache, sinks = attend_steps(gpu, FULL)
    run([1, 1, 1, 1, 1, 1], 6)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        torch.full((1 << 24,), float("nan"), device=gpu)
    first.replay()
    rows = 64
    qkv = torch.randn(rows, cache.cfg.qkv_width, device=gpu, dtype=torch.bfloat16)
    new = i32([1, 2, 3, 4, 5, 6], gpu)
    with torch.cuda.graph(second, pool=first.pool()):
        cache.step = table.step(new, rows)
        got = cache.attend(qkv, sinks)
    assert (run([1, 0, 1, 0, 0, 0], rows)[2:] == 0).all()
    second.replay()
    assert (got[:21] != 0).any() and (got[21:] == 0).all()
    assert (run([1, 0, 1, 0, 0, 0], rows)[2:] == 0).all()
    cache.step.check()


def test_padding_rows_of_a_paged_stack_stay_finite(gpu):
    from mimo_moe.paged import PagedDecoderStack
    stack = PagedDecoderStack(stack_layers(gpu), max_requests=3, max_len=256, num_pages=40, page_size=16)
    x = torch.randn(40, 1024, device=gpu).to(torch.bfloat16)
    x[30:] = float("nan")
    assert torch.isnan(stack(x, i32([20, 10, 10], gpu))[30:]).all()
    x = torch.zeros(40, 1024, device=gpu, dtype=torch.bfloat16)
    assert torch.isfinite(stack(x, i32([1, 1, 0], gpu))).all()
    stack.check()


def test_rope_store_paged_refuses_another_clear(gpu):
    from mimo_moe import paged
    cfg = cfg_of(D64)
    step, _, N = layout([0], [4], 16, gpu, 2)
    cache = paged.PagedKVCache(cfg, N, 16, gpu)
    qkv = torch.zeros(4, cfg.qkv_width, dtype=torch.bfloat16, device=gpu)
    good = torch.zeros(4, cfg.n_heads, cfg.v_head_dim, dtype=torch.bfloat16, device=gpu)
    paged.rope_store_paged(qkv, cfg, cache, step, clear=good)
    for bad in (good[:3], good.float(), good.cpu(), good[:, :4], torch.zeros(4, 16, 64, dtype=torch.bfloat16,
                                                                             device=gpu)[:, ::2]):
        with pytest.raises(ValueError):
            paged.rope_store_paged(qkv, cfg, cache, step, clear=bad)


def test_a_plan_of_earlier_lengths_is_refused_until_it_is_made_again(gpu):
    """A step planned again in place, and a step whose table has gone on: the attention plan of the lengths before."""
    from mimo_moe import paged
    cfg, P, N = cfg_of(D64), 16, 40
    lens, free = i32([0, 0], gpu), torch.arange(N, dtype=torch.int32, device=gpu)
    table = torch.full((2, 8), -1, dtype=torch.int32, device=gpu)
    cache = paged.PagedKVCache(cfg, N, P, gpu)
    gen = torch.Generator(gpu).manual_seed(3)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, generator=gen, device=gpu))
    q = torch.randn(40, cfg.n_heads, cfg.head_dim, generator=gen, device=gpu).to(torch.bfloat16)
    step = paged.page_plan(lens, i32([30, 10], gpu), table, free, i32([N], gpu), P, 40)
    plan = paged.attention_plan(step, cfg)
    first = paged.attention_paged(q, cache, cfg, step, plan=plan)
    paged.page_plan(lens, i32([7, 33], gpu), table, free, i32([N], gpu), P, 40, out=step)
    with pytest.raises(ValueError, match="update"):
        paged.attention_paged(q, cache, cfg, step, plan=plan)
    want = paged.attention_paged(q, cache, cfg, step)
    plan.update()
    assert torch.equal(paged.attention_paged(q, cache, cfg, step, plan=plan), want) and not torch.equal(first, want)
    # steps of one table
    pages = paged.PageTable(2, 128, N, P, gpu)
    one = pages.step(i32([3, 4], gpu), 7)
    plan = paged.attention_plan(one, cfg)
    paged.attention_paged(q[:7], cache, cfg, one, plan=plan)
    two = pages.step(i32([1, 1], gpu), 7)
    with pytest.raises(ValueError, match="update"):
        paged.attention_paged(q[:7], cache, cfg, one, plan=plan)
    paged.attention_paged(q[:7], cache, cfg, two, plan=paged.attention_plan(two, cfg))
    none = pages.step(i32([0, 0], gpu), 0)
    paged.attention_paged(q[:0], cache, cfg, none, plan=paged.attention_plan(none, cfg))
    # captured: the plan is made again inside the graph, which then serves any lengths
    new, left = i32([30, 10], gpu), i32([N], gpu)
    plan = paged.attention_plan(step, cfg)
    out = torch.zeros(40, cfg.n_heads, cfg.v_head_dim, dtype=torch.bfloat16, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.page_plan(lens, new, table, free, left, P, 40, out=step)
        plan.update()
        paged.attention_paged(q, cache, cfg, step, plan=plan, out=out)
    for lengths, expect in (([30, 10], first), ([7, 33], want)):
        new.copy_(i32(lengths, gpu))
        graph.replay()
        assert torch.equal(out, expect)
    step.check()


@pytest.mark.parametrize("blocks", [200, 1500, 2100, 40_000], ids=lambda b: f"{b} blocks")
def test_how_long_units_are_dealt_goes_by_their_lengths_alone(gpu, blocks):
    """Whole or split (another order of a row's sum) is the same however often a plan is made and whichever request has
    which length.  Two units for each SM, 20 of them two blocks longer than the others: a CTA that gets two of the 20 makes
    splitting worth it, one that gets one does not, so an order that is left to chance shows."""
    from mimo_moe import paged
    cfg, P = cfg_of(dict(D64, n_heads=1, n_kv_heads=1)), 128
    R = 2 * torch.cuda.get_device_properties(gpu).multi_processor_count
    lens = [128 * (blocks + 2 * (r < 20)) for r in range(R)]
    table = torch.zeros(R, max(lens) // P, dtype=torch.int32, device=gpu)
    rng, modes = np.random.default_rng(blocks), []
    for order in [list(range(R)), list(range(R))[::-1]] + [rng.permutation(R).tolist() for _ in range(16)]:
        rows = torch.zeros(R, dtype=torch.int32, device=gpu)
        step = paged.PageStep(block_table=table, page_size=P, cu_q=i32(list(range(R + 1)), gpu),
                              seq_lens=i32([lens[r] for r in order], gpu), positions=rows, slots=rows)
        for _ in range(3):
            plan = paged.attention_plan(step, cfg)
            head = plan.buffer[:12].view(torch.int32).tolist()
            assert head[1] == R
            modes.append(head[2])
        step.check()
    assert len(set(modes)) == 1, modes
