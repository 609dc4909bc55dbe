"""Attention over a paged key-value cache against its definition in 64 bits: one new token a sequence, and the last tokens of
ragged batches."""
import math
import random
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


@pytest.fixture(scope="module")
def paged():
    from oracle import paged_oracle

    return paged_oracle


def make(dev, lens, new=None, heads=8, kv=2, dim=64, page=16, dtype=torch.bfloat16, seed=0, spare=3, columns=0, tail=0, scale=1.0):
    """Query, caches, table, lengths and starts (None for one token a sequence).  Places behind a sequence's end hold NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    need = [max(0, -(-n // page)) for n in lens]
    pages = sum(need) + spare
    width = max(need + [columns])
    ids = list(range(pages))
    rng.shuffle(ids)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.full((pages, page, kv, dim), math.nan, dtype=dtype, device=dev)
    v = torch.full_like(k, math.nan)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = ids.pop()
            rows = min(page, n - i * page)
            k[table[b, i], :rows] = torch.randn((rows, kv, dim), generator=g, device=dev).to(dtype)
            v[table[b, i], :rows] = torch.randn((rows, kv, dim), generator=g, device=dev).to(dtype)
    starts, tokens = None, len(lens)
    if new is not None:
        starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
        tokens = sum(new) + tail
    q = (torch.randn((tokens, heads, dim), generator=g, device=dev) * scale).to(dtype)
    return q, k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), starts


def call(npu, q, k, v, table, lens, starts, **kw):
    if starts is None:
        return npu.npu_paged_attention(q, k, v, table, lens, **kw)
    return npu.npu_paged_prompt_attention(q, k, v, table, lens, starts, **kw)


def check(npu, paged, q, k, v, table, lens, starts, **kw):
    out, lse = call(npu, q, k, v, table, lens, starts, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    assert lse.shape == q.shape[:2] and lse.dtype == torch.float32
    kw = {"scale": kw.pop("scale_value", None), **kw}
    ref = paged.attention(q, k, v, table, lens, starts, **kw)
    bound, lse_bound = paged.attention_bounds(q.dtype, q.shape[2], *ref)
    none = ref[1] == -math.inf
    assert torch.equal(lse == -math.inf, none) and bool((out[none] == 0).all())
    err = (out.double() - ref[0]).abs()
    assert bool((err <= bound).all()), f"out is off by {(err / bound).nan_to_num(nan=math.inf).max().item():.2f} times its bound"
    err = (lse.double() - ref[1])[~none].abs()
    assert bool((err <= lse_bound[~none]).all()), f"lse is off by {(err / lse_bound[~none]).max().item():.2f} times its bound"
    return out, lse


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 72, 80, 128, 200, 256])
def test_decode_head_dimensions(npu, paged, dev, dim, dtype):
    check(npu, paged, *make(dev, LENS, dim=dim, dtype=dtype, seed=dim))


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (7, 1), (12, 4), (16, 1), (34, 2), (32, 1), (40, 1)])
def test_decode_groups(npu, paged, dev, heads, kv):
    check(npu, paged, *make(dev, LENS, heads=heads, kv=kv, dim=128, seed=heads))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 100, 128, 512])
def test_decode_page_sizes(npu, paged, dev, page):
    check(npu, paged, *make(dev, LENS, page=page, dim=128, seed=page))


WINDOWS = [(1, 0), (1, 1), (7, 0), (16, 4), (33, 40), (64, 5), (100, 129), (128, 1), (1000, 4), (2**31, 2**31)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_decode_window(npu, paged, dev, window, sinks):
    check(npu, paged, *make(dev, LENS + [1000], dim=128, seed=window % 97), window=window, sinks=sinks)


def test_decode_long(npu, paged, dev):
    """Split over the cache's length and joined; one sequence among short ones."""
    check(npu, paged, *make(dev, [20011], heads=8, kv=2, dim=128, seed=1))
    check(npu, paged, *make(dev, [3, 9000, 0, 40, 4097], heads=4, kv=4, dim=64, seed=2))
    check(npu, paged, *make(dev, [20011], heads=8, kv=2, dim=128, seed=3), window=9000, sinks=70)


def test_decode_many_sequences(npu, paged, dev):
    rng = random.Random(5)
    check(npu, paged, *make(dev, [rng.choice([0, 1, rng.randrange(60)]) for _ in range(1500)], heads=2, kv=1, dim=64, seed=4))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 8.0])
def test_decode_scales(npu, paged, dev, scale):
    check(npu, paged, *make(dev, LENS, dim=64, seed=8), scale_value=scale)


NEW = [(1, 1), (2, 2), (17, 17), (1, 300), (5, 133), (130, 130), (64, 128), (0, 50), (3, 2), (0, 0), (129, 400), (260, 261)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 72, 80, 128, 200, 256])
def test_prompt_head_dimensions(npu, paged, dev, dim, dtype):
    check(npu, paged, *make(dev, [n for _, n in NEW], [n for n, _ in NEW], dim=dim, dtype=dtype, seed=dim, tail=3))


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (7, 1), (12, 4), (16, 1), (34, 2), (32, 1), (130, 1)])
def test_prompt_groups(npu, paged, dev, heads, kv):
    check(npu, paged, *make(dev, [n for _, n in NEW], [n for n, _ in NEW], heads=heads, kv=kv, dim=128, seed=heads))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 100, 128, 512])
def test_prompt_page_sizes(npu, paged, dev, page):
    check(npu, paged, *make(dev, [n for _, n in NEW], [n for n, _ in NEW], page=page, dim=128, seed=page))


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_prompt_window(npu, paged, dev, window, sinks):
    lens, new = [n for _, n in NEW] + [900], [n for n, _ in NEW] + [700]
    check(npu, paged, *make(dev, lens, new, dim=128, seed=window % 97), window=window, sinks=sinks)


def test_prompt_few_tokens_long_cache(npu, paged, dev):
    """Few rows: split over the cache's length and joined."""
    check(npu, paged, *make(dev, [20011], [4], heads=8, kv=2, dim=128, seed=1))
    check(npu, paged, *make(dev, [30, 9000, 0, 40, 4097], [2, 3, 0, 1, 5], heads=4, kv=4, dim=64, seed=2))
    check(npu, paged, *make(dev, [20011], [7], heads=8, kv=2, dim=256, seed=3), window=9000, sinks=70)


def check_rows(npu, paged, q, k, v, table, lens, starts, count, **kw):
    """check() for some of many rows."""
    out, lse = call(npu, q, k, v, table, lens, starts, **kw)
    only = set(random.Random(1).sample(range(q.shape[0]), count)) | {0, q.shape[0] - 1}
    ref = paged.attention(q, k, v, table, lens, starts, only=only, **kw)
    bound, lse_bound = paged.attention_bounds(q.dtype, q.shape[2], *ref)
    rows = torch.tensor(sorted(only), device=q.device)
    assert bool(((out.double() - ref[0]).abs() <= bound)[rows].all())
    none = ref[1] == -math.inf
    assert torch.equal((lse == -math.inf)[rows], none[rows])
    assert bool(((lse.double() - ref[1]).abs() <= lse_bound)[rows][~none[rows]].all())
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("heads,kv,dim,page", [(32, 8, 128, 16), (20, 4, 128, 64), (28, 4, 64, 128), (16, 16, 96, 24), (16, 2, 256, 32),
                                               (64, 1, 128, 16), (12, 4, 256, 7)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3)])
def test_prompt_more_items_than_the_gpu_takes_at_once(npu, paged, dev, heads, kv, dim, page, window, sinks):
    """CTAs that go on from item to item: one row tile and two, odd and even numbers of steps, items without any."""
    rng = random.Random(dim + heads)
    new = [rng.choice([0, 1, 3, rng.randrange(30), rng.randrange(300)]) for _ in range(90)] + [1000]
    lens = [max(0, n + rng.choice([0, 0, -2, rng.randrange(40), rng.randrange(700)])) for n in new]
    check_rows(npu, paged, *make(dev, lens, new, heads=heads, kv=kv, dim=dim, page=page, seed=heads, tail=2), 150, window=window, sinks=sinks)


def test_decode_large_batch(npu, paged, dev):
    rng = random.Random(9)
    lens = [rng.choice([rng.randrange(700), rng.randrange(3000)]) for _ in range(300)]
    check_rows(npu, paged, *make(dev, lens, heads=32, kv=8, dim=128, seed=1), 60)
    check_rows(npu, paged, *make(dev, lens, heads=40, kv=2, dim=64, seed=2), 60, window=500, sinks=5)


def test_tokens_before_the_first_and_behind_the_last(npu, paged, dev):
    """Rows of no sequence in front and behind, and a sequence that has pages of another one, whose prefix it shares."""
    q, k, v, table, lens, starts = make(dev, [200, 200, 90], [40, 40, 0], dim=128, seed=21, tail=60)
    table[1, :10] = table[0, :10]
    check(npu, paged, q, k, v, table, lens, starts + 7)
    check(npu, paged, q[:3], k, v, table, lens, None)
    q, k, v, table, lens, starts = make(dev, [20011, 100], [4, 2], heads=8, kv=2, dim=128, seed=22, tail=3)  # split
    check(npu, paged, q, k, v, table, lens, starts + 2)


@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 16, 2), (256, 4, 2), (80, 12, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2500, 4)])
def test_pieces_of_ragged_sequences(npu, paged, dev, dim, heads, kv, window, sinks):
    """Few tokens: long sequences are cut, short ones are not, some see nothing; short ones alone in a table that could hold
    much; what a captured graph does when the lengths change."""
    rng = random.Random(dim)
    lens, new = [20011, 100, 0, 5000, 17, -3, 9000, 2], [3, 2, 2, 40, 1, 1, 0, 4]
    check(npu, paged, *make(dev, lens, new, heads=heads, kv=kv, dim=dim, seed=25, tail=3), window=window, sinks=sinks)
    state = make(dev, [90, 33, 1, 128], [4, 3, 1, 2], heads=heads, kv=kv, dim=dim, seed=26, columns=3000)
    check(npu, paged, *state, window=window, sinks=sinks)
    lens = [rng.randrange(20, 6000) for _ in range(12)]
    q, k, v, table, lens, starts = make(dev, lens, [rng.randrange(1, 7) for _ in lens], heads=heads, kv=kv, dim=dim, seed=27)
    graph = torch.cuda.CUDAGraph()
    call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)
    for change in (lambda n: n, lambda n: (n // 50).clamp(min=1), lambda n: n * 0, lambda n: n.roll(3).minimum(n)):
        kept = lens.clone()
        lens.copy_(change(lens))
        graph.replay()
        want = call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
        ref = paged.attention(q, k, v, table, lens, starts, window=window, sinks=sinks)
        bound, lse_bound = paged.attention_bounds(q.dtype, dim, *ref)
        assert bool(((got[0].double() - ref[0]).abs() <= bound).all())
        none = ref[1] == -math.inf
        assert torch.equal(got[1] == -math.inf, none) and bool(((got[1].double() - ref[1]).abs() <= lse_bound)[~none].all())
        lens.copy_(kept)


@pytest.mark.parametrize("dim", [128, 256])
def test_values_not_finite_where_a_row_is_split(npu, paged, dev, dim):
    """As above for a few tokens over a long cache, whose parts are added by another kernel."""
    for window, sinks in ((0, 0), (3000, 3)):
        q, k, v, table, lens, starts = make(dev, [9000, 5000], [6, 5], heads=8, kv=2, dim=dim, seed=23)
        ref = paged.attention(q, k, v, table, lens, starts, window=window, sinks=sinks)
        bound = paged.attention_bounds(q.dtype, dim, *ref)[0]
        for b, j in ((0, 8997), (0, 5997), (1, 4998), (1, 1)):
            v2 = v.clone()
            v2[table[b, j // 16], j % 16, 0, 3] = math.nan
            out, _ = call(npu, q, k, v2, table, lens, starts, window=window, sinks=sinks)
            rows = paged.rows_of(lens.tolist(), starts.tolist(), q.shape[0])
            hit = torch.zeros_like(out, dtype=torch.bool)
            hit[:, :4, 3] = torch.tensor([s == b and j <= p and (window == 0 or p - j < window or j < sinks) for s, p in rows], device=dev)[:, None]
            assert bool(out[hit].isnan().all()) and bool(((out.double() - ref[0]).abs() <= bound)[~hit].all()), (window, b, j)


def test_prompt_many_sequences(npu, paged, dev):
    rng = random.Random(6)
    new = [rng.choice([0, 1, rng.randrange(9)]) for _ in range(700)]
    check(npu, paged, *make(dev, [n + rng.choice([0, 0, rng.randrange(40)]) for n in new], new, heads=2, kv=1, dim=64, seed=4))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 8.0])
def test_prompt_scales(npu, paged, dev, scale):
    check(npu, paged, *make(dev, [n for _, n in NEW], [n for n, _ in NEW], dim=64, seed=8), scale_value=scale)


def _both(dev, **kw):
    yield make(dev, LENS, **kw)
    yield make(dev, [n for _, n in NEW], [n for n, _ in NEW], **kw)


def test_large_scores(npu, paged, dev):
    """Scores of some hundreds: one key takes all the weight, the running maximum moves by much."""
    for a in _both(dev, dim=128, scale=30.0, seed=11):
        check(npu, paged, *a)


def test_scores_that_grow_along_the_cache(npu, paged, dev):
    """Every block of keys has larger scores than the one before it, by more and by less than what moves the base."""
    for step in (0.01, 0.2, 3.0):
        for q, k, v, table, lens, starts in _both(dev, dim=64, seed=12):
            place = torch.zeros(k.shape[:2], device=dev)
            for b, row in enumerate(table.tolist()):
                for i, page in enumerate(row):
                    if page >= 0:
                        place[page] = torch.arange(i * 16, i * 16 + 16, device=dev)
            k[..., 0] = (place * step).to(k.dtype)[..., None]
            q[..., 0] = 1.0
            check(npu, paged, q, k, v, table, lens, starts)


def test_strides_and_layouts(npu, paged, dev):
    """Query rows from a fused projection, heads in front of places in the cache, a table with spare columns between rows."""
    for q, k, v, table, lens, starts in _both(dev, dim=128, seed=13):
        T, H, D = q.shape
        fused = torch.randn((T, 3 * H * D), device=dev).to(q.dtype)
        fused[:, H * D:2 * H * D] = q.reshape(T, -1)
        wide = torch.full((table.shape[0], 2 * table.shape[1] + 3), 7, dtype=torch.int32, device=dev)
        wide[:, :table.shape[1]] = table
        want = call(npu, q, k, v, table, lens, starts)
        kh = k.transpose(1, 2).contiguous().transpose(1, 2)
        vh = torch.full((v.shape[0] * 2, *v.shape[1:]), math.nan, device=dev, dtype=v.dtype)[::2]
        vh.copy_(v)
        got = call(npu, fused[:, H * D:2 * H * D].view(T, H, D), kh, vh, wide[:, :table.shape[1]], lens, starts)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
        # what the vectors cannot reach: copied for the query
        odd = torch.zeros(q.numel() + 1, device=dev, dtype=q.dtype)[1:].view(q.shape)
        odd.copy_(q)
        got = call(npu, odd, k, v, table.t().contiguous().t(), lens, starts)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_bad_pages_and_lengths(npu, paged, dev):
    """Pages outside the cache are not seen; lengths behind the table's end see what it covers; negative ones see nothing."""
    for q, k, v, table, lens, starts in _both(dev, dim=64, seed=14):
        bad = table.clone()
        flat = bad.view(-1)
        flat[::3] = torch.tensor([-1, k.shape[0], 2**31 - 1, -2**31], device=dev, dtype=torch.int32).repeat(flat.numel())[:flat[::3].numel()]
        check(npu, paged, q, k, v, bad, lens, starts)
        check(npu, paged, q, k, v, bad[:, :5], lens, starts)
        check(npu, paged, q, k, v, table[:, :0], lens, starts)
        check(npu, paged, q, k[:0], v[:0], table, lens, starts)
        if starts is None:
            lens = lens.clone()
            lens[3::4] = torch.tensor([-1, -2**31, -7, 0], device=dev, dtype=torch.int32)[:lens[3::4].numel()]
            check(npu, paged, q, k, v, table, lens, starts)
    q, k, v, table, lens, starts = make(dev, [40, 50], [20, 20], seed=15)
    check(npu, paged, q, k, v, table, torch.tensor([-5, 2**31 - 1], dtype=torch.int32, device=dev)[:1].repeat(2), starts)
    check(npu, paged, q, k, v, table, torch.tensor([-2**31, 50], dtype=torch.int32, device=dev), starts)


def test_nothing_unseen_is_read(npu, paged, dev):
    """NaN and infinities in places that a token does not see, behind it and behind its window, change nothing in its row."""
    for poison in (math.nan, math.inf, -math.inf):
        for q, k, v, table, lens, starts in _both(dev, dim=128, seed=16):
            window, sinks = 40, 3
            want = call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)
            k2, v2 = k.clone(), v.clone()
            for b, n in enumerate(lens.tolist()):
                new = 1 if starts is None else int(starts[b + 1] - starts[b])
                for j in range(sinks, n - new - window + 1):
                    k2[table[b, j // 16], j % 16] = poison
                    v2[table[b, j // 16], j % 16] = poison
            got = call(npu, q, k2, v2, table, lens, starts, window=window, sinks=sinks)
            assert torch.equal(want[1], got[1])
            if starts is None:
                assert torch.equal(want[0], got[0])
            else:  # a prompt's rows that came beside such values are made again, in another order
                ref = paged.attention(q, k, v, table, lens, starts, window=window, sinks=sinks)
                assert bool(((got[0].double() - ref[0]).abs() <= paged.attention_bounds(q.dtype, 128, *ref)[0]).all())


@pytest.mark.parametrize("dim,page", [(128, 16), (128, 128), (64, 64), (256, 48), (96, 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 0), (200, 5), (1, 140)])
def test_what_is_behind_a_sequence(npu, paged, dev, dim, page, window, sinks):
    """The rest of the last page holds anything and changes no bit; pages that a window has left may be other sequences' or gone."""
    for split in (False, True):
        lens, new = ([6000, 5003], [5, 3]) if split else ([700, 333, 128, 41], [300, 333, 60, 41])
        q, k, v, table, lens, starts = make(dev, lens, new, dim=dim, page=page, seed=24)
        want = call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)
        ref = paged.attention(q, k, v, table, lens, starts, window=window, sinks=sinks)
        assert bool(((want[0].double() - ref[0]).abs() <= paged.attention_bounds(q.dtype, dim, *ref)[0]).all())
        k2, v2, table2 = k.clone(), v.clone(), table.clone()
        for b, n in enumerate(lens.tolist()):
            for j in range(n, -(-n // page) * page):
                k2[table[b, j // page], j % page] = math.nan
                v2[table[b, j // page], j % page] = math.nan
            low = n - int(starts[b + 1] - starts[b]) - window + 1  # the first token's window
            if window > 0:
                for i in range(-(-sinks // page), max(0, low) // page):
                    table2[b, i] = (-1, 1 << 30, int(table[1 - min(b, 1), 0]))[i % 3]
        got = call(npu, q, k2, v2, table2, lens, starts, window=window, sinks=sinks)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_values_not_finite_reach_their_rows_alone(npu, paged, dev, poison):
    """A value that is not finite, at places in the middle of a prompt: rows before it, and rows whose window has passed it,
    are as they were; rows that see it are not finite."""
    for window, sinks in ((0, 0), (50, 2), (200, 140)):
        q, k, v, table, lens, starts = make(dev, [300, 280], [290, 280], dim=128, seed=17)
        lse_want = call(npu, q, k, v, table, lens, starts, window=window, sinks=sinks)[1]
        ref = paged.attention(q, k, v, table, lens, starts, window=window, sinks=sinks)
        bound = paged.attention_bounds(q.dtype, 128, *ref)[0]
        for b, j in ((0, 0), (0, 1), (0, 131), (1, 127), (1, 200)):
            v2 = v.clone()
            v2[table[b, j // 16], j % 16, 1, 5:9] = poison
            out, lse = call(npu, q, k, v2, table, lens, starts, window=window, sinks=sinks)
            assert torch.equal(lse, lse_want)
            rows = paged.rows_of(lens.tolist(), starts.tolist(), q.shape[0])
            sees = torch.tensor([s == b and j <= p and (window == 0 or p - j < window or j < sinks) for s, p in rows], device=dev)
            hit = torch.zeros_like(out, dtype=torch.bool)
            hit[:, 4:, 5:9] = sees[:, None, None]
            assert bool((~out[hit].isfinite()).all()), (window, sinks, b, j)
            assert bool(((out.double() - ref[0]).abs() <= bound)[~hit].all()), (window, sinks, b, j)


def test_keys_not_finite(npu, paged, dev):
    """A key that is NaN makes the rows that see it NaN, and no other."""
    q, k, v, table, lens, starts = make(dev, [300, 280], [290, 280], dim=64, seed=18)
    want = call(npu, q, k, v, table, lens, starts, window=60, sinks=1)
    j = 140
    k2 = k.clone()
    k2[table[0, j // 16], j % 16, 0, 3] = math.nan
    out, lse = call(npu, q, k2, v, table, lens, starts, window=60, sinks=1)
    rows = paged.rows_of(lens.tolist(), starts.tolist(), q.shape[0])
    sees = torch.tensor([s == 0 and j <= p and p - j < 60 for s, p in rows], device=dev)
    assert bool(sees.any()) and bool(out[sees][:, :4].isnan().all()) and bool(lse[sees][:, :4].isnan().all())
    assert torch.equal(out[~sees], want[0][~sees]) and torch.equal(out[:, 4:], want[0][:, 4:]) and torch.equal(lse[~sees], want[1][~sees])


def test_results_do_not_change_from_call_to_call(npu, dev):
    for a in (make(dev, [5000, 70, 1], dim=128), make(dev, [5000, 300], [4, 299], dim=128), make(dev, [2000, 900], [1500, 900], dim=128)):
        first = call(npu, *a)
        for _ in range(5):
            again = call(npu, *a)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_graphs_and_streams(npu, dev):
    """Two graphs captured one after the other, replayed at the same time on two streams with new lengths and tables."""
    for a in (make(dev, [3000, 900], dim=128), make(dev, [3000, 900], [5, 3], dim=128), make(dev, [700, 900], [600, 900], dim=128)):
        q, k, v, table, lens, starts = a
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(npu, *a)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs, inputs = [], [], []
        for i in range(2):
            inputs.append([t.clone() if t is not None else None for t in a])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(call(npu, *inputs[i]))
            graphs.append(g)
        for i in range(2):
            inputs[i][0].copy_(q * (1 + i))
            inputs[i][4].copy_(lens - 17 * i)
        want = [call(npu, *inputs[i]) for i in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(10):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


def test_offsets_beyond_32_bits(npu, paged, dev):
    """Pages that lie more than 2^31 elements into the cache."""
    pages, page, kv, dim = 140000, 16, 8, 128  # 2.3e9 elements a cache
    k = torch.empty((pages, page, kv, dim), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    for lens, new in (([70, 33], None), ([70, 33], [50, 3])):
        q, ks, vs, table, length, starts = make(dev, lens, new, heads=16, kv=kv, dim=dim, seed=19)
        far = torch.where(table >= 0, pages - 1 - table, table)
        k[pages - ks.shape[0]:] = ks.flip(0)
        v[pages - vs.shape[0]:] = vs.flip(0)
        want = call(npu, q, ks, vs, table, length, starts)
        got = call(npu, q, k, v, far, length, starts)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_prompt_of_one_token_is_decode(npu, paged, dev):
    a = make(dev, [5, 300, 77], [1, 1, 1], dim=128, seed=20)
    check(npu, paged, *a[:5], None)
    check(npu, paged, *a)


def test_empty_calls(npu, dev):
    q, k, v, table, lens, starts = make(dev, [5], [5])
    out, lse = npu.npu_paged_attention(q[:0], k, v, table[:0], lens[:0])
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    out, lse = npu.npu_paged_prompt_attention(q[:0], k, v, table[:0], lens[:0], starts[:1])
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    out, lse = npu.npu_paged_prompt_attention(q, k, v, table[:0], lens[:0], starts[:1])
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, lse = npu.npu_paged_attention(q[:1, :0], k, v, table, lens)
    assert out.shape == (1, 0, 64) and lse.shape == (1, 0)


def test_refusals(npu, dev):
    q, k, v, table, lens, starts = make(dev, [5, 9], [2, 3])
    one = q[:2]

    def refused(text, *a, **kw):
        f = npu.npu_paged_prompt_attention if len(a) == 6 else npu.npu_paged_attention
        with pytest.raises(RuntimeError, match=text):
            f(*a, **kw)

    refused("bfloat16 or float16", one.float(), k.float(), v.float(), table, lens)
    refused("dtype of the query", one, k.half(), v, table, lens)
    refused("same shape", one, k, v[:-1], table, lens)
    refused("page size", one, k[0], v, table, lens)
    refused("multiple of the cache's", one[:, :3], k, v, table, lens)
    refused("same head dimension", one[..., :32], k, v, table, lens)
    refused("last dimension", one, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, lens)
    refused("int32", one, k, v, table.long(), lens)
    refused("int32", one, k, v, table, lens.long())
    refused("int32", one, k, v, table, lens[:1])
    refused("one token for each", q, k, v, table, lens)
    refused("not be negative", one, k, v, table, lens, window=-1)
    refused("not be negative", one, k, v, table, lens, window=3, sinks=-1)
    refused("with a window only", one, k, v, table, lens, sinks=4)
    refused("finite", one, k, v, table, lens, scale_value=math.inf)
    refused("finite", one, k, v, table, lens, scale_value=math.nan)
    refused("int32 \\[3\\]", q, k, v, table, lens, starts[:2])
    refused("int32", q, k, v, table, lens, starts.long())
    refused("should be on", one, k.cpu(), v, table, lens)
    refused("should be on", one, k, v, table.cpu(), lens)
    refused("should be on", q, k, v, table, lens, starts.cpu())
    wide = torch.zeros((4, 16, 2, 68), dtype=q.dtype, device=dev)
    refused("multiples of 8", one, wide[..., :64], wide[..., :64], table, lens)
    refused("multiple of 8", one[..., :12].contiguous(), k[..., :12].contiguous(), v[..., :12].contiguous(), table, lens)
    big = torch.zeros((2, 2, 264), dtype=q.dtype, device=dev)
    refused("up to 256", big, big[:, :, None].expand(2, 2, 2, 264).contiguous(), big[:, :, None].expand(2, 2, 2, 264).contiguous(), table, lens)
