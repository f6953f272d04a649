"""The attention block on the 4-bit cache without a device: what its entry points refuse, its
sizes, the page tables of Kv4Cache, and the 64-bit reference of the GPU tests against the
layout that the header describes."""
import ctypes as C

import pytest
import torch

import iree_amd
import kv4ref
from iree_amd import flags as F

ONE = C.c_void_p(4096)
ODD = C.c_void_p(4096 + 8)
T = F.ATTENTION_TYPE_F16


def _call(name, defaults, **changes):
    lib = iree_amd.load_library()
    return getattr(lib, "iree_amd_uk_" + name)(*{**defaults, **changes}.values())


ROPE = dict(q=ONE, q_stride=512, k=ONE, k_stride=256, v=ONE, v_stride=256, q_out=ONE, q_out_stride=512, k_out=ONE,
            k_out_stride=256, q_weight=ONE, k_weight=ONE, eps=1e-6, cos_sin=ONE, table_rows=10, rotary=128, positions=ONE,
            cache=ONE, pages=4, page_stride=2 * 16 * 136, page_size=16, slots=ONE, tokens=3, heads=4, kv_heads=2,
            dim=128, flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=3)), (3, dict(flags=T | 0x200)), (12, dict(dim=96)), (3, dict(dim=-64)),
    (3, dict(tokens=-1)), (3, dict(tokens=1 << 31)), (3, dict(heads=-4)), (3, dict(kv_heads=-1)),
    (3, dict(eps=-1.0)), (3, dict(eps=float("nan"))), (3, dict(rotary=4)), (3, dict(rotary=136)), (3, dict(rotary=20)),
    (3, dict(table_rows=-1)), (3, dict(page_size=24)), (3, dict(page_size=8)), (3, dict(page_size=512)),
    (3, dict(pages=-1)), (3, dict(pages=1 << 31)), (3, dict(page_stride=2 * 16 * 136 - 16)),
    (3, dict(page_stride=2 * 16 * 136 + 8)), (3, dict(cache=ODD)), (3, dict(page_stride=1 << 62)),
    (3, dict(q_out=None)), (3, dict(k=None)), (3, dict(v=None)), (3, dict(slots=None)), (3, dict(positions=None)),
    (3, dict(q_stride=504)), (3, dict(k_stride=248)), (3, dict(v_stride=-256)), (3, dict(k_out_stride=128)),
    (3, dict(cache=None)), (3, dict(cache=None, v=None, k_out=None)),
    (12, dict(q=ODD)), (12, dict(k_out=ODD)), (12, dict(v_stride=260)), (12, dict(q_weight=ODD)), (12, dict(cos_sin=ODD)),
    (3, dict(q_stride=1024)), (3, dict(k_stride=264)),      # in place (q_out is q here) with another stride
])
def test_norm_and_rotation_refuse(status, changes):
    assert _call("qk_norm_rope", ROPE, **changes) == status
    assert iree_amd.load_library().iree_amd_uk_last_error()


def test_norm_and_rotation_of_nothing():
    nothing = dict(q=None, k=None, v=None, cache=None)
    assert _call("qk_norm_rope", ROPE, tokens=0) == 0
    assert _call("qk_norm_rope", ROPE, **nothing) == 0
    assert _call("qk_norm_rope", ROPE, heads=0, kv_heads=0) == 0


READ = dict(cache=ONE, pages=4, page_stride=2 * 16 * 72, page_size=16, slots=ONE, k_out=ONE, k_stride=128, v_out=ONE,
            v_stride=128, rows=3, kv_heads=2, dim=64, flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=T | 0x100)), (12, dict(dim=32)), (3, dict(rows=-1)), (3, dict(cache=None)),
    (3, dict(slots=None)), (3, dict(k_stride=120)), (12, dict(v_out=ODD)), (3, dict(page_size=17)),
    (3, dict(page_stride=16)),
])
def test_read_refuses(status, changes):
    assert _call("kv4_read", READ, **changes) == status


def test_read_of_nothing():
    assert _call("kv4_read", READ, rows=0) == 0
    assert _call("kv4_read", READ, k_out=None, v_out=None) == 0


ATTENTION = dict(q=ONE, q_stride=512, out=ONE, out_stride=512, cache=ONE, pages=4, page_stride=2 * 16 * 136, page_size=16,
                 page_table=ONE, table_stride=2, max_pages=2, q_starts=ONE, kv_lens=ONE, tokens=3, batch=3, heads=4,
                 kv_heads=2, dim=128, scale=0.1, window=0, sinks=0, max_kv_len=32, workspace=None, workspace_bytes=0,
                 flags=T, stream=None)


@pytest.mark.parametrize("status,changes", [
    (3, dict(flags=0)), (3, dict(flags=T | 0x100)), (12, dict(dim=80)), (3, dict(heads=5)), (3, dict(kv_heads=0)),
    (3, dict(heads=1 << 17, kv_heads=1)), (3, dict(tokens=-1)), (3, dict(batch=-1)), (3, dict(window=-1)),
    (3, dict(sinks=-1)), (3, dict(max_kv_len=-1)), (3, dict(table_stride=1)), (3, dict(max_pages=-1)),
    (3, dict(page_table=None)), (3, dict(q_starts=None)), (3, dict(kv_lens=None)), (3, dict(cache=None)),
    (3, dict(scale=float("inf"))), (3, dict(scale=float("nan"))), (3, dict(q=None)), (3, dict(out=None)),
    (3, dict(q_stride=504)), (12, dict(out_stride=516)), (12, dict(q=ODD)), (3, dict(workspace_bytes=64)),
    (3, dict(workspace=ODD, workspace_bytes=64)), (3, dict(page_size=33)), (3, dict(page_stride=0)),
])
def test_attention_refuses(status, changes):
    assert _call("attention_kv4", ATTENTION, **changes) == status


def test_attention_refuses_positions_past_31_bits():
    most = (2**31 - 4096) // 256
    at = dict(page_size=256, page_stride=2 * 256 * 136)
    assert _call("attention_kv4", ATTENTION, max_pages=most + 1, table_stride=most + 1, **at) == 3
    assert _call("attention_kv4", ATTENTION, max_pages=most, table_stride=most, q=None, **at) == 3      # (that q is null)
    assert b"null q" in iree_amd.load_library().iree_amd_uk_last_error()


def test_attention_of_nothing():
    for empty in (dict(tokens=0), dict(batch=0), dict(heads=0)):
        assert _call("attention_kv4", ATTENTION, **empty) == 0
    assert iree_amd.attention_kv4_workspace(0, 4, 8, 2, 128, max_kv_len=1 << 20) == 0
    with pytest.raises(iree_amd.UkError):
        iree_amd.attention_kv4_workspace(1, 1, 3, 2, 128, max_kv_len=10)
    with pytest.raises(iree_amd.UkError):
        iree_amd.attention_kv4_workspace(1, 1, 2, 2, 120, max_kv_len=10)


@pytest.mark.parametrize("status,src,dst,changes", [
    (11, [0, 4], [1, 2], {}), (11, [0, -1], [1, 2], {}), (11, [0, 1], [2, 4], {}), (11, [0], [-2], {}),
    (3, [0, 1], [2, 2], {}), (3, [0, 1], [2, 0], {}), (3, [1], [1], {}), (3, [0], [1], dict(page_bytes=40)),
    (3, [0], [1], dict(stride=16)), (3, [0], [1], dict(stride=72)), (3, [0], [1], dict(pages=-1)),
    (3, [0], [1], dict(count=-1)), (3, [0], [1], dict(pool=ODD)), (3, [0], [1], dict(pool=None)),
])
def test_copy_pages_refuses(status, src, dst, changes):
    s, d = (torch.tensor(x, dtype=torch.int32) for x in (src, dst))
    args = dict(pool=ONE, pages=4, page_bytes=48, stride=64, src=s.data_ptr(), dst=d.data_ptr(), count=len(src), stream=None)
    assert _call("copy_pages", args, **changes) == status
    assert _call("copy_pages", {**args, "count": 0}) == 0


def test_wrappers_refuse_other_tensors():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        iree_amd.qk_norm_rope(x, None, x, None, 4, 1, 0, 64, T)
    with pytest.raises(ValueError):
        iree_amd.copy_pages(x, 4, 16, [0], [1, 2])
    with pytest.raises(ValueError):
        iree_amd.copy_pages(x, 4, 16, torch.tensor([0]), torch.tensor([1]))


def test_page_bytes():
    assert iree_amd.kv4_page_bytes(16, 8, 128) == 8 * 16 * 136
    assert iree_amd.kv4_page_bytes(256, 0, 64) == 0
    for bad in ((24, 1, 64), (16, -1, 64), (16, 1, 65)):
        with pytest.raises(iree_amd.UkError):
            iree_amd.kv4_page_bytes(*bad)


def test_the_reference_packs_as_the_header_says():
    """Byte by byte, from the header's words."""
    gen = torch.Generator().manual_seed(4)
    pages, heads, page, dim = 2, 3, 16, 64
    k, v = (torch.randn(pages, heads, page, dim, generator=gen).half() for _ in range(2))
    cache = kv4ref.pack(k, v, page)
    assert cache.shape == (pages, heads * page * (dim + 8))
    kc, vc, kp, vp = kv4ref.load(cache, page, heads, dim)
    for rows, codes, params in ((k, kc, kp), (v, vc, vp)):
        c, s, m = kv4ref.quantise(rows)
        assert torch.equal(codes, c.double()) and torch.equal(params, torch.stack((s, m), -1).double())
    for p, h, t, d in ((0, 0, 0, 0), (1, 2, 15, 63), (1, 1, 6, 37), (0, 2, 9, 8)):
        block = cache[p, h * page * (dim + 8):(h + 1) * page * (dim + 8)].tolist()
        assert (block[t * dim // 2 + d // 2] >> 4 * (d % 2)) & 15 == kc[p, h, t, d]
        dword = (t // 4 * (dim // 8) + d // 8) * 4 + t % 4
        assert (block[page * dim // 2 + dword * 4 + d % 8 // 2] >> 4 * (d % 2)) & 15 == vc[p, h, t, d]
    # values stand within half a step of the row, and for constants exactly
    c, s, m = kv4ref.quantise(k)
    assert bool(((c * s.double()[..., None] + m.double()[..., None] - k.double()).abs() <=
                 s.double()[..., None] * 0.5 * (1 + 16 * 2.0**-10)).all())
    c, s, m = kv4ref.quantise(torch.full((1, 64), 0.3).half())
    assert not c.any() and s == 0 and m == torch.tensor(0.3).half()


def _pool(monkeypatch, pages=8, page=16):
    from iree_amd import attention
    copies = []

    def record(buffer, total, nbytes, src, dst):
        copies.extend(zip(src, dst))
        buffer[torch.tensor(dst)] = buffer[torch.tensor(src)]

    monkeypatch.setattr(attention, "copy_pages", record)
    pool = iree_amd.Kv4Cache(pages, page, 2, 1, 64, device="cpu")
    return pool, copies


def test_cache_extends_and_ends_sequences(monkeypatch):
    pool, _ = _pool(monkeypatch)
    a, b = pool.new(), pool.new()
    slots = pool.extend([a, b], [17, 3]).tolist()
    assert len(set(slots)) == 20 and pool.free_pages() == 5
    table, lens, wide = pool.tables([b, a])
    assert lens.tolist() == [3, 17] and wide == 2 and table.tolist()[0][1] == -1
    assert [table[1, t // 16] * 16 + t % 16 for t in range(17)] == slots[:17]
    assert pool.extend([a], [0]).numel() == 0
    with pytest.raises(MemoryError):
        pool.extend([b, a], [14, 80])
    assert pool.free_pages() == 5 and pool.length(a) == 17 and pool.length(b) == 3
    for bad in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1])):
        with pytest.raises(ValueError):
            pool.extend(*bad)
    pool.extend([b, a], [13, 64])
    assert pool.free_pages() == 1
    pool.free(a)
    pool.free(b)
    assert pool.free_pages() == 8
    with pytest.raises(KeyError):
        pool.free(a)


def test_cache_forks_share_full_pages(monkeypatch):
    pool, copies = _pool(monkeypatch)
    a = pool.new()
    pool.extend([a], [32])
    b = pool.fork(a)
    assert not copies and pool.free_pages() == 6
    pool.extend([a], [1])
    c = pool.fork(a)
    assert len(copies) == 1 and pool.free_pages() == 4
    pool.extend([b, c], [1, 1])
    own = [pool.tables([s])[0][0, 2].item() for s in (a, b, c)]
    assert len(set(own)) == 3 and pool.free_pages() == 3
    pool.free(a)
    assert pool.free_pages() == 4
    pool.free(b)
    pool.free(c)
    assert pool.free_pages() == 8
    e = pool.fork(pool.new())
    assert pool.length(e) == 0
    full = pool.new()
    pool.extend([full], [8 * 16 - 1])
    with pytest.raises(MemoryError):
        pool.fork(full)
    assert pool.free_pages() == 0 and len(copies) == 1


def test_cache_drops_what_no_later_token_sees(monkeypatch):
    pool, _ = _pool(monkeypatch)
    a = pool.new()
    pool.extend([a], [100])
    # token 100 sees those from 100 - window + 1 on, and the first `sinks`
    pool.drop(a, 21, sinks=17)          # from 80: pages 2, 3 and 4 end at or before it, 0 and 1 hold sinks
    assert [p < 0 for p in pool.tables([a])[0][0].tolist()] == [False, False, True, True, True, False, False]
    pool.drop(a, 21, sinks=0)
    assert [p < 0 for p in pool.tables([a])[0][0].tolist()] == [True] * 5 + [False, False]
    assert pool.free_pages() == 6
    pool.drop(a, 1000)
    b = pool.fork(a)
    pool.extend([a], [12])
    pool.drop(a, 1)
    assert pool.tables([a])[0][0].tolist() == [-1] * 7
    pool.extend([a], [1])
    with pytest.raises(ValueError):
        pool.drop(a, 0)
    pool.free(a)
    pool.free(b)
    assert pool.free_pages() == 8


def test_cache_compacts(monkeypatch):
    pool, copies = _pool(monkeypatch)
    seqs = [pool.new() for _ in range(6)]
    for i, s in enumerate(seqs):
        for slot in pool.extend([s], [16]).tolist():
            pool.buffer[slot // 16] = i + 1
    twin = pool.fork(seqs[5])
    for s in (seqs[0], seqs[2], seqs[3]):
        pool.free(s)
    assert pool.compact() == 3
    table = pool.tables([seqs[1], seqs[4], seqs[5], twin])[0][:, 0].tolist()
    assert sorted(table[:3]) == [0, 1, 2] and table[2] == table[3]
    assert [int(pool.buffer[p, 0]) for p in table] == [2, 5, 6, 6]
    assert len(copies) == 2 and pool.free_pages() == 5
    assert pool.compact() == 3 and len(copies) == 2
    assert sorted(pool.extend([seqs[1]], [80]).tolist()) == list(range(48, 128))


@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(32768, 32, 8, 128), (131072, 32, 8, 128), (524288, 32, 8, 64),
                                                       (131072, 16, 4, 256), (1 << 20, 8, 8, 256)])
def test_long_prompts_ask_for_a_bounded_workspace(tokens, heads, kv_heads, dim):
    assert 0 < iree_amd.attention_kv4_workspace(tokens, 1, heads, kv_heads, dim, max_kv_len=tokens) <= 256 << 20
    assert iree_amd.attention_kv4_workspace(tokens, 1, heads, kv_heads, dim, max_kv_len=tokens, window=50000) <= 256 << 20
    # (one tile of 128 rows of every head, in 64 parts, is more)
    most = max(256 << 20, kv_heads * 64 * 128 * (dim + 2) * 4)
    assert iree_amd.attention_kv4_workspace(tokens, 1, heads, kv_heads, dim, max_kv_len=1 << 20) <= most


def test_the_workspace_query_refuses_a_length_it_cannot_know():
    """0 is the page table's capacity for the call; the query, which has no page table, took it for one key."""
    with pytest.raises(iree_amd.UkError):
        iree_amd.attention_kv4_workspace(2, 2, 8, 2, 128, max_kv_len=0)
    assert b"max_kv_len" in iree_amd.load_library().iree_amd_uk_last_error()
    assert iree_amd.attention_kv4_workspace(2, 2, 8, 2, 128, max_kv_len=1) == 0
    assert iree_amd.attention_kv4_workspace(0, 2, 8, 2, 128, max_kv_len=0) == 0
