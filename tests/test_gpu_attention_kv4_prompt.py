"""attention_kv4 on prompts that fill the device, against its formula in 64 bits."""
import math

import pytest
import torch

import kv4ref
from test_gpu_attention_kv4 import BF16, F16, Case, _gen, _normal

pytestmark = pytest.mark.gpu


def _replace(case, k, v):
    """Rows [pages][kv heads][page][D] in place of the case's own, what no sequence owns still NaN."""
    old = case.cache.view(case.pages, case.kv_heads, -1)
    new = kv4ref.pack(k, v, case.page).view(old.shape)
    at = case.page * case.dim
    unowned = (old[..., at:] == 0xFF)
    new[..., at:][unowned] = 0xFF
    old.copy_(new)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_lens", [(4, 2, [3, 40]), (64, 16, [130, 128, 200, 150])])
def test_values_past_the_range_of_f16(uk, cuda, heads, kv_heads, q_lens, dim, window, sinks):
    """V rows of bf16 whose offset + 8 scales pass 65504, as far as both saturate: finite in the
    result of the queries that see them, without a trace in that of all others, before them and behind
    their window."""
    case = Case(61, BF16, heads, kv_heads, dim, 16, q_lens, [n + 70 for n in q_lens])
    gen = _gen(62)
    k, v = (_normal(gen, case.pages, kv_heads, 16, dim) for _ in range(2))
    k, v = k.to(BF16), v.to(BF16)
    ramp = torch.linspace(0, 1, dim, device="cuda")
    for token, row in ((33, ramp * 150000), (75, ramp * 1e30), (76, (ramp - 1) * 1e30), (90, 60000 + ramp * 9e4),
                       (101, (ramp - 0.5) * 3e38)):
        for b, n in enumerate(case.kv_lens):
            if token < n:
                v[int(case.table[b, token // 16]), :, token % 16] = row.to(BF16)
    _replace(case, k, v)
    out = case.run(uk, window=window, sinks=sinks)
    assert bool(torch.isfinite(out).all())
    case.check(out, window=window, sinks=sinks)


# (batches whose rows come to the prompt kernel's 128 a sequence, and to work for a whole device: kv heads times
# tiles of 128 rows, or these times tiles of 64 keys)
WIDE = (64, 16, [130, 128, 200, 150])


def _taken(uk, split=False):
    assert uk.last_kernel_path() == "attention_kv4:prompt" + ("-split" if split else "")


@pytest.mark.parametrize("heads,kv_heads,dim,page,q_lens,kv_lens,path", [
    (32, 8, 128, 16, [1, 1], [40, 300], "attention_kv4:few-rows"),
    (4, 2, 128, 16, [3, 40], [73, 110], "attention_kv4:few-rows"),
    (32, 8, 64, 64, [1, 1], [20000, 40], "attention_kv4:few-rows-split"),
    (64, 16, 256, 16, [130, 128, 200, 150], [200, 198, 270, 220], "attention_kv4:few-rows"),
    (64, 16, 128, 16, [130, 128, 200, 150], [200, 198, 270, 220], "attention_kv4:prompt"),
    (64, 16, 64, 16, [130, 128, 200, 150], [200, 198, 270, 220], "attention_kv4:prompt"),
    (8, 2, 128, 64, [300], [30000], "attention_kv4:prompt-split")])
def test_the_kernel_that_is_taken(uk, cuda, heads, kv_heads, dim, page, q_lens, kv_lens, path):
    case = Case(1, F16, heads, kv_heads, dim, page, q_lens, kv_lens)
    case.check(case.run(uk))
    assert uk.last_kernel_path() == path


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 256), (128, 32), (128, 128)])
@pytest.mark.parametrize("heads,kv_heads,q_lens,kv_lens", [
    (*WIDE, [130, 300, 200, 1001]),
    (40, 40, [150, 0, 300, 77, 129], [150, 80, 901, 77, 512]),
    (36, 12, [700, 333], [700, 340]),
    (130, 2, [700, 1, 2], [777, 1, 90])])
def test_prompts(uk, cuda, dtype, heads, kv_heads, dim, page, q_lens, kv_lens):
    """Whole prompts, continued ones, single tokens and an empty sequence beside them; 1, 3, 4 and 65 query
    heads to a kv head."""
    case = Case(dim + heads, dtype, heads, kv_heads, dim, page, q_lens, kv_lens)
    case.check(case.run(uk))
    _taken(uk)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (31, 33), (40, 0), (64, 64), (100, 70), (129, 200),
                                          (999, 4), (1 << 50, 1 << 50)])
def test_windows_and_sinks(uk, cuda, dim, window, sinks):
    case = Case(window % 97 + sinks % 89, F16 if sinks % 2 else BF16, *WIDE[:2], dim, 32, WIDE[2], [130, 333, 700, 150])
    case.check(case.run(uk, window=window, sinks=sinks), window=window, sinks=sinks)
    _taken(uk)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_lens", [[0, 5, -3, 100], [129, 64, 200, 1]])
def test_rows_that_see_nothing_are_zero(uk, cuda, dim, kv_lens):
    case = Case(5, F16, *WIDE[:2], dim, 16, WIDE[2], kv_lens)
    out = case.run(uk)
    _taken(uk)
    case.check(out)
    for b, (n, kv) in enumerate(zip(case.q_lens, kv_lens)):
        empty = out[case.starts[b]:case.starts[b] + max(0, n - max(kv, 0)), :case.heads * dim]
        assert bool((empty == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_pages_that_do_not_exist(uk, cuda, dim):
    """Entries of -1 and beyond the pool hide their tokens, a whole sequence's too, with and without a window."""
    missing = [(0, 1, -1), (0, 4, 1 << 30), (1, 0, -7), (3, 9, -1), (3, 10, -1), (3, 11, -1)]
    missing += [(2, i, -1) for i in range(17)]
    case = Case(11, BF16, *WIDE[:2], dim, 16, WIDE[2], [150, 190, 270, 290], missing=missing)
    for window, sinks in ((0, 0), (50, 20)):
        out = case.run(uk, window=window, sinks=sinks)
        _taken(uk)
        case.check(out, window=window, sinks=sinks)
        assert bool((out[case.starts[2]:case.starts[3], :case.heads * dim] == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_rows_that_are_not_finite(uk, cuda, dim, which):
    """A cached row that was not finite makes NaN of every query that sees it and of no other: not of
    earlier ones in its tile, nor of those whose window has passed it."""
    case = Case(17, F16, *WIDE[:2], dim, 16, WIDE[2], [210, 200, 230, 300])
    kv_heads = case.kv_heads
    view = case.cache.view(case.pages, kv_heads, -1)
    at = 16 * dim if which == "keys" else 16 * (dim + 4)
    for token in (150, 197):
        page = int(case.table[0, token // 16])
        view[page, 1, at + token % 16 * 4:at + token % 16 * 4 + 4] = torch.tensor([0, 0x7E, 0, 0], dtype=torch.uint8)
    q_len = case.q_lens[0]
    position = torch.arange(q_len, device="cuda") + 210 - q_len
    for window, sinks in ((0, 0), (30, 0), (30, 151)):
        out = case.run(uk, window=window, sinks=sinks)
        _taken(uk)
        bad = torch.isnan(out[case.starts[0]:case.starts[1], :64 * dim]).view(q_len, 16, 4, dim)
        sees = torch.zeros_like(position, dtype=torch.bool)
        for token in (150, 197):
            sees |= (position >= token) & ((position < token + window) | (window == 0) | (token < sinks))
        assert bool(bad[:, 1][sees].all()) and not bool(bad[:, 1][~sees].any())
        assert not bool(bad[:, [0] + list(range(2, 16))].any())
        assert not bool(torch.isnan(out[case.starts[1]:case.starts[4]]).any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size,scale", [(30.0, None), (1e-4, 2.0), (1.0, 0.0), (1.0, -0.3), (2000.0, 1e-3)])
def test_sizes_of_scores(uk, cuda, dtype, dim, size, scale):
    """Scores that leave one key, that are all but equal, negative scales."""
    case = Case(21, dtype, *WIDE[:2], dim, 32, WIDE[2], [333, 200, 270, 150], size=size)
    case.check(case.run(uk, scale=scale), scale=scale)
    _taken(uk)


@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_of_values(uk, cuda, dim):
    """V rows from 2^-20 to 2^14, zeros and constants among them, in one sequence."""
    case = Case(31, F16, *WIDE[:2], dim, 16, WIDE[2], [400, 200, 210, 333])
    gen = _gen(3)
    shape = (case.pages, case.kv_heads, 16, dim)
    v = _normal(gen, *shape) * 2.0 ** torch.randint(-20, 14, (*shape[:3], 1), generator=gen, device="cuda")
    v[:, :, 3] = 0
    v[:, :, 7] = 1.5
    _replace(case, _normal(gen, *shape).half(), v.half())
    case.check(case.run(uk))
    _taken(uk)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20000, 77)])
@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 128), (F16, 64)])
def test_next_parts_of_prompts_are_split(uk, cuda, dtype, dim, window, sinks):
    """Long cached prefixes: the call with the workspace it asks for, the same bits twice, with too
    little, and with a wrong idea of the lengths."""
    q_lens, kv_lens = [450, 300], [30000, 26011]
    case = Case(12, dtype, 8, 2, dim, 64, q_lens, kv_lens)
    nbytes = uk.attention_kv4_workspace(case.tokens, 2, 8, 2, dim, max_kv_len=30000, window=window, sinks=sinks)
    assert nbytes > 0
    workspace = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    more = dict(window=window, sinks=sinks)
    first = case.run(uk, max_kv_len=30000, workspace=workspace, **more)
    _taken(uk, split=True)
    case.check(first, **more)
    workspace.fill_(0x7F)
    assert torch.equal(first, case.run(uk, max_kv_len=30000, workspace=workspace, **more))
    case.check(case.run(uk, max_kv_len=30000, workspace=workspace[:64], **more), **more)
    _taken(uk)
    case.check(case.run(uk, max_kv_len=25000, **more), **more)
    _taken(uk, split=True)


def test_sequences_of_no_rows_between_prompts(uk, cuda):
    """More sequences than a wave looks at in one step."""
    q_lens = [2100 if b % 13 == 6 else 0 for b in range(130)]
    case = Case(6, BF16, 32, 8, 128, 16, q_lens, [b % 50 + n for b, n in enumerate(q_lens)])
    case.check(case.run(uk))
    _taken(uk)


def test_captured_and_replayed(uk, cuda):
    """Two graphs of prompts, one of them split, replayed in turns with eager calls between."""
    cases = [Case(40, F16, *WIDE[:2], 128, 16, WIDE[2], [300, 400, 500, 600]),
             Case(41, F16, 8, 2, 128, 64, [450, 300], [30000, 26011])]
    graphs, outs = [], []
    for case, split in zip(cases, (False, True)):
        case.run(uk)
        _taken(uk, split)
        out = torch.full((case.tokens, case.heads * 128 + 16), 3.0, dtype=F16, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            case.run(uk, out=out)
        graphs.append(graph)
        outs.append(out)
    for turn in range(3):
        for case, graph, out in zip(cases, graphs, outs):
            case.q.mul_(-0.7)
            case.device_lens.sub_(41)
            case.kv_lens = [n - 41 for n in case.kv_lens]
            out.fill_(3.0)
            graph.replay()
        eager = [case.run(uk) for case in cases]
        torch.cuda.synchronize()
        for case, out, want in zip(cases, outs, eager):
            assert torch.equal(out, want)
    cases[0].check(outs[0])


def test_two_calls_at_once(uk, cuda):
    cases = [Case(50 + i, F16, 8, 2, 128, 64, [450, 300], [30000 - 999 * i, 7000]) for i in range(2)]
    want = [case.run(uk) for case in cases]
    _taken(uk, split=True)
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.full_like(w, 3.0) for _ in range(4)] for w in want]
    torch.cuda.synchronize()
    for turn in range(4):
        for case, stream, mine in zip(cases, streams, outs):
            case.run(uk, out=mine[turn], stream=stream)
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for w, mine in zip(want, outs) for out in mine)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,q_lens", [(8, 2, [1, 5]), WIDE])
def test_a_key_of_all_the_weight_with_small_values(uk, cuda, dtype, dim, heads, kv_heads, q_lens):
    """One key whose score is far above the others' and whose V row is 2^-28 of theirs: the weights keep
    their bits next to what they are multiplied with."""
    case = Case(33, dtype, heads, kv_heads, dim, 16, q_lens, [n + 150 for n in q_lens])
    case.q.abs_()
    gen = _gen(34)
    shape = (case.pages, kv_heads, 16, dim)
    k, v = _normal(gen, *shape), _normal(gen, *shape).clamp(-3, 3) * 2.0**14
    for b in range(len(q_lens)):
        page = int(case.table[b, 2])
        k[page, :, 9] = 300 / dim
        v[page, :, 9] *= 2.0**-28
    _replace(case, k.half(), v.half())
    case.check(case.run(uk, scale=0.13), scale=0.13)
    if dim < 256:
        assert uk.last_kernel_path() == "attention_kv4:" + ("prompt" if q_lens is WIDE[2] else "few-rows")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,q_lens,kv_lens", [(64, 8, [1] * 8, [300, 1000, 20000, 77, 4000, 513, 900, 65]),
                                                           (*WIDE, [130, 500, 2000, 150])])
def test_results_are_off_by_their_own_rounding(uk, cuda, dtype, dim, heads, kv_heads, q_lens, kv_lens):
    """A rounding to a type is off evenly within half a step: by step^2 / 12 in the mean square. Over 32768 results
    and more that mean is within 3 % (5 / sqrt(32768)) of it, and f32 scores and sums, at 2^-24 times a few hundred
    (bf16: an f16 weight, whose 2^-11 is squared 1/64 of the result's 2^-8), leave the rest of a tenth. One f16 weight
    a key would come to twice as much with results of f16."""
    case = Case(71, dtype, heads, kv_heads, dim, 64, q_lens, kv_lens)
    out = case.run(uk)
    q = case.q[:, :heads * dim].reshape(case.tokens, heads, dim)
    want, _ = kv4ref.attention(q, case.cache, 64, case.table[:, :case.wide], case.starts, kv_lens, kv_heads,
                               case.scale(None))
    got = out[case.rows][:, :heads * dim].double()
    want = want[case.rows].reshape(got.shape)
    step = torch.exp2(torch.frexp(want)[1].double()) * torch.finfo(dtype).eps / 2
    assert float((got - want).square().mean()) < 1.1 * float(step.square().mean()) / 12


@pytest.mark.parametrize("heads,kv_heads,dim,q_lens", [(64, 16, 128, [2500, 1700]), (64, 16, 256, [1100, 1000])])
def test_prompts_whose_partial_results_are_many(uk, cuda, heads, kv_heads, dim, q_lens):
    """More partial results than a call asks memory for: several launches use the same. Rows from all over both
    sequences, the last row of each among them, against the formula; all rows against the call without memory."""
    kv_lens = [33000, 20000]
    case = Case(81, F16, heads, kv_heads, dim, 64, q_lens, kv_lens)
    nbytes = uk.attention_kv4_workspace(case.tokens, 2, heads, kv_heads, dim, max_kv_len=max(kv_lens))
    tile = 128 if dim <= 128 else 16      # rows; 33000 keys are split in 3 at least
    assert (case.tokens * 4 // tile + 2) * kv_heads * 3 * tile * (dim + 2) * 4 > 256 << 20 >= nbytes
    workspace = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    out = case.run(uk, max_kv_len=max(kv_lens), workspace=workspace)
    assert uk.last_kernel_path() == "attention_kv4:" + ("prompt" if dim <= 128 else "few-rows") + "-split"
    assert bool((out[~case.rows] == 3).all()) and bool((out[:, heads * dim:] == 3).all())
    plain = case.run(uk, max_kv_len=max(kv_lens), workspace=workspace[:64])
    assert "split" not in uk.last_kernel_path()
    a, b = out[case.rows][:, :heads * dim].double(), plain[case.rows][:, :heads * dim].double()
    # (each within half a step and what f32 sums of 33000 keys come to)
    assert bool(((a - b).abs() <= 2.0**-10 * b.abs() + 2.0**-10 * 0.05).all())
    for s, (q_len, kv_len) in enumerate(zip(q_lens, kv_lens)):
        token = torch.tensor(sorted({0, 1, 31, 32, q_len // 3, q_len // 2 + 5, q_len - 33, q_len - 1}), device="cuda")
        rows = case.starts[s] + token
        q = case.q[rows][:, :heads * dim].reshape(len(token), heads, dim)
        table = case.table[s:s + 1, :case.wide].expand(len(token), -1)
        want, bound = kv4ref.attention(q, case.cache, 64, table, list(range(len(token) + 1)),
                                       [kv_len - q_len + int(t) + 1 for t in token], kv_heads, case.scale(None))
        kv4ref.assert_near(out[rows][:, :heads * dim].reshape(want.shape), want, bound)


def test_no_idea_of_the_lengths_is_the_capacity(uk, cuda):
    """0 and None split a long cache alike, with the memory that the call takes for itself."""
    case = Case(91, F16, 8, 2, 128, 64, [1, 1], [40000, 33])
    want = case.run(uk)
    assert uk.last_kernel_path() == "attention_kv4:few-rows-split"
    assert torch.equal(want, case.run(uk, max_kv_len=0))
    assert uk.last_kernel_path() == "attention_kv4:few-rows-split"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_lens,wide", [(8, 2, [1, 5], 3), (*WIDE, 9)])
def test_tokens_past_the_page_table_are_not_seen(uk, cuda, heads, kv_heads, q_lens, wide, dim):
    """Lengths that pass max_pages pages, in the middle of a tile."""
    case = Case(95, F16, heads, kv_heads, dim, 16, q_lens, [n + 60 for n in q_lens])
    case.wide = wide
    for window, sinks in ((0, 0), (33, 5)):
        case.check(case.run(uk, window=window, sinks=sinks), window=window, sinks=sinks)
        assert uk.last_kernel_path() == "attention_kv4:" + ("prompt" if wide == 9 else "few-rows")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_lens", [(8, 2, [1, 5]), WIDE])
def test_scores_of_any_size_are_finite(uk, cuda, heads, kv_heads, q_lens, dim):
    """Queries of 2^90, or 2^-100: of scores that lie so far apart one key has all of the weight; of scores of 0 all
    keys have the same. (A weight in f16 is within 2^-11 of itself, of V rows whose 15 scales and offset come to less
    than 8.)"""
    case = Case(97, BF16, heads, kv_heads, dim, 32, q_lens, [n + 60 for n in q_lens])
    case.q.mul_(2.0**88)
    for _ in range(2):
        out = case.run(uk)
        q = case.q[:, :heads * dim].reshape(case.tokens, heads, dim)
        want, _ = kv4ref.attention(q, case.cache, 32, case.table[:, :case.wide], case.starts, case.kv_lens, kv_heads,
                                   case.scale(None))
        got = out[:, :heads * dim].reshape(want.shape)
        assert bool(torch.isfinite(got[case.rows]).all())
        kv4ref.assert_near(got, want, torch.full_like(want, 2.0**-11 * 8), rows=case.rows)
        case.q.mul_(2.0**-95).mul_(2.0**-95)
