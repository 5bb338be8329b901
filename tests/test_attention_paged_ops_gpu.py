"""Prompt and single-token attention over caller-owned pages
(ndl_attention_prompt, ndl_attention_split) against 64 bits, within bounds
derived in paged_support.bound."""
import numpy as np
import pytest
import torch

from paged_support import TYPES, Cache, attend, bound

pytestmark = pytest.mark.gpu


def _i32(a, cuda):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=cuda)


def _queries(cache, kind, rows, heads, cuda, size=1.0):
    q = torch.from_numpy(size * cache.rng.normal(size=(rows, heads, 64))).to(TYPES[kind])
    return q.to(cuda), q.double().numpy()


def _check(kind, got, cache, slot, q, position, window, scale=0.125):
    """One row's output [heads, 64] against 64 bits."""
    keys, values = cache.keys(slot), cache.values(slot)
    out, size, reach = attend(q, keys, values, position, window, scale)
    seen = min(position + 1, window) if window else position + 1
    limit = bound(kind, out, size, reach, max(seen, 0), np.abs(values).max() if len(values) else 0.0)
    got = got.double().cpu().numpy()
    off = np.abs(got - out)
    if kind == "f16":  # 65520 and above round to infinity
        off[(got == np.copysign(np.inf, out)) & (np.abs(out) + limit >= 65520.0)] = 0.0
    assert np.all(off <= limit), (slot, position, window, (off / limit).max())


# ------------------------------------------------------------ single tokens --

@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (4, 1), (6, 2), (15, 3), (16, 1), (34, 2), (2, 2)])
def test_split_matches_64_bits(ops, cuda, kind, heads, kv_heads):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 0, 511, 700]
    cache = Cache(heads + kv_heads, lengths, kv_heads)
    slots = list(cache.rng.permutation(len(lengths)))
    q, x = _queries(cache, kind, len(slots), heads, cuda)
    for window in (0, 1, 40, 64, 257):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = ops.attention_split(q, _i32(slots, cuda), _i32([lengths[s] for s in slots], cuda), kv_heads,
                                  *cache.device(cuda), window=window, status=status)
        assert status.item() == 0 and out.dtype == TYPES[kind]
        for r, s in enumerate(slots):
            _check(kind, out[r], cache, s, x[r], lengths[s] - 1, window)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,heads,kv_heads,window", [(1, 8, 8, 0), (24, 34, 2, 0), (33, 6, 3, 0), (148, 4, 1, 0),
                                                        (149, 4, 1, 0), (1, 4, 2, 800), (36, 34, 2, 100), (49, 3, 3, 1)])
def test_split_of_short_rows(ops, cuda, kind, rows, heads, kv_heads, window):
    """Short slots, or a short window of long ones, as many items as SMs and one more: no row reads more than 16
    pages."""
    rng = np.random.default_rng(rows + heads)
    lengths = [int(n) for n in rng.integers(0, 1500 if window else 1025, rows)]
    cache = Cache(rows, lengths, kv_heads, spare_columns=0)
    if not window:
        assert cache.max_pages <= 16
    q, x = _queries(cache, kind, rows, heads, cuda)
    out = ops.attention_split(q, _i32(range(rows), cuda), _i32(lengths, cuda), kv_heads, *cache.device(cuda), window=window)
    for r, n in enumerate(lengths):
        _check(kind, out[r], cache, r, x[r], n - 1, window)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,length", [(1, 20000), (2, 9001), (3, 4097), (9, 2050)])
def test_split_of_long_rows(ops, cuda, kind, rows, length):
    lengths = [length - 37 * r for r in range(rows)]
    cache = Cache(rows, lengths, 2, layers=1, layer=0)
    q, x = _queries(cache, kind, rows, 8, cuda, size=3.0)
    for window in (0, 3000):
        out = ops.attention_split(q, _i32(range(rows), cuda), _i32(lengths, cuda), 2, *cache.device(cuda),
                                  window=window)
        for r in range(rows):
            _check(kind, out[r], cache, r, x[r], lengths[r] - 1, window)


def test_split_of_many_rows(ops, cuda):
    """More (row, head) pairs than thread blocks, several rows on one slot."""
    cache = Cache(1, [5, 900, 64, 333], 4, layers=1, layer=0)
    rows = 700
    slots = cache.rng.integers(0, 4, rows)
    lens = [int(cache.rng.integers(0, cache.lengths[s] + 1)) for s in slots]
    q, x = _queries(cache, "bf16", rows, 8, cuda)
    out = ops.attention_split(q, _i32(slots, cuda), _i32(lens, cuda), 4, *cache.device(cuda))
    for r in range(0, rows, 7):
        _check("bf16", out[r], cache, slots[r], x[r], lens[r] - 1, 0)


@pytest.mark.parametrize("kind", list(TYPES))
def test_split_peaked_scores_and_extreme_scales(ops, cuda, kind):
    """One position far above the rest, value scales over 60 binary orders, and zero scales."""
    lengths = [200, 333]
    cache = Cache(17, lengths, 2, layers=1, layer=0, peak=8.0)
    for s in range(2):
        cache.vs[s][:] = 2.0 ** cache.rng.integers(-30, 30, cache.vs[s].shape)
        cache.vs[s][::7] = 0.0
        cache.ks[s][::5] = 0.0
    _repack(cache)
    q, x = _queries(cache, kind, 2, 4, cuda)
    out = ops.attention_split(q, _i32([0, 1], cuda), _i32(lengths, cuda), 2, *cache.device(cuda))
    for r in range(2):
        _check(kind, out[r], cache, r, x[r], lengths[r] - 1, 0)
    rows = sum(lengths)
    q, x = _queries(cache, kind, rows, 4, cuda)
    out = ops.attention_prompt(q, _i32([0, 200, 533], cuda), _i32([0, 1], cuda), _i32([0, 0], cuda), 2,
                               *cache.device(cuda))
    for r in (0, 1, 50, 199, 200, 263, 264, 532):
        s = r >= 200
        _check(kind, out[r], cache, int(s), x[r], r - 200 * s, 0)


def _repack(cache):
    """The cache's arrays into its pool again."""
    from attention_support import K_BYTE, K_OFF, KS_OFF, S_SLOT, V_BYTE, V_OFF, VS_OFF

    for s, n in enumerate(cache.lengths):
        for i in range((n + 63) // 64):
            lo, hi = i * 64, min(n, i * 64 + 64)
            c = hi - lo
            for h in range(cache.kv_heads):
                rec = cache.pool[cache.table[s, i], cache.layer, h]
                rec[K_OFF + K_BYTE[:c]] = cache.k[s][lo:hi, h].view(np.uint8)
                rec[V_OFF + V_BYTE[:c]] = cache.v[s][lo:hi, h].view(np.uint8)
                rec[KS_OFF:KS_OFF + 256].view(np.float32)[S_SLOT[:c]] = cache.ks[s][lo:hi, h]
                rec[VS_OFF:VS_OFF + 256].view(np.float32)[:c] = cache.vs[s][lo:hi, h]


@pytest.mark.parametrize("kind", list(TYPES))
def test_large_and_tiny_queries(ops, cuda, kind):
    """Queries near the type's ends: the scores come out of range only where 64 bits' do."""
    cache = Cache(21, [90], 1, layers=1, layer=0)
    big = {"f32": 1e30, "f16": 3e4, "bf16": 1e30}[kind]
    q, x = _queries(cache, kind, 4, 2, cuda)
    factors = [0.0, 2.0 ** -20, 1.0, 2.0 ** 6]
    q = q * torch.tensor(factors, dtype=q.dtype, device=cuda)[:, None, None]
    x = q.double().cpu().numpy()
    out = ops.attention_split(q, _i32([0] * 4, cuda), _i32([90] * 4, cuda), 1, *cache.device(cuda))
    for r in range(4):
        _check(kind, out[r], cache, 0, x[r], 89, 0)
    # a scale that brings huge queries back to ordinary scores
    unit = torch.ones_like(q) * (q.abs() > 0)
    q2 = (torch.sign(q) * unit * big).to(q.dtype)
    scale = float(np.float32(0.5 / big))
    args = (_i32([0] * 4, cuda), _i32([90] * 4, cuda), 1, *cache.device(cuda))
    out = ops.attention_split(q2, *args, scale=scale)
    x = q2.double().cpu().numpy()
    for r in range(1, 4):
        _check(kind, out[r], cache, 0, x[r], 89, 0, scale=scale)
    out = ops.attention_prompt(q2, _i32([0, 4], cuda), _i32([0], cuda), _i32([80], cuda), 1, *cache.device(cuda),
                               scale=scale)
    for r in range(1, 4):
        _check(kind, out[r], cache, 0, x[r], 80 + r, 0, scale=scale)


def test_split_strided_rows_and_given_outputs(ops, cuda):
    cache = Cache(23, [100, 40, 900], 2)
    qkv = torch.randn((3, 4 * 64 + 2 * 2 * 64), device=cuda).to(torch.bfloat16)
    q = qkv[:, :256].unflatten(1, (4, 64))
    args = (_i32([2, 0, 1], cuda), _i32([900, 100, 40], cuda), 2, *cache.device(cuda))
    want = ops.attention_split(q.contiguous(), *args)
    wide = torch.full((3, 512), 5.0, device=cuda, dtype=torch.bfloat16)
    got = ops.attention_split(q, *args, out=wide[:, 128:384].unflatten(1, (4, 64)))
    assert torch.equal(got, want)
    assert torch.all(wide[:, :128] == 5.0) and torch.all(wide[:, 384:] == 5.0)


def test_split_bad_rows(ops, cuda):
    """Bad slots, lengths and pages: NaN for that row alone, status 2."""
    lengths = [100, 200, 3000, 64]
    cache = Cache(25, lengths, 2)
    good = ops.attention_split(*_split_args(cache, [0, 1, 2, 3], lengths, cuda))
    cache.table[2, 40] = cache.num_pages
    cache.table[1, 1] = -7
    rows = [(0, 100), (4, 10), (-1, 10), (2, 3000), (2, 64 * 40), (1, 200), (1, 64), (3, -1),
            (3, 64 * cache.max_pages + 1), (3, 64)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    args = _split_args(cache, [s for s, _ in rows], [n for _, n in rows], cuda)
    q0 = _split_args(cache, [0, 1, 2, 3], lengths, cuda)[0]
    q = args[0]
    q[0], q[9] = q0[0], q0[3]
    out = ops.attention_split(*args, status=status)
    assert status.item() == 2
    nan = torch.isnan(out).flatten(1)
    assert nan.all(1).tolist() == [False, True, True, True, False, True, False, True, True, False]
    assert not nan[[0, 4, 6, 9]].any()
    assert torch.equal(out[0], good[0]) and torch.equal(out[9], good[3])


def _split_args(cache, slots, lens, cuda):
    rng = np.random.default_rng(99)
    q = torch.from_numpy(rng.normal(size=(len(slots), 4, 64))).half().to(cuda)
    return (q, _i32(slots, cuda), _i32(lens, cuda), 2, *cache.device(cuda))


@pytest.mark.parametrize("what", ["k", "v", "q"])
def test_nan_stays_in_its_head(ops, cuda, what):
    """A NaN scale or query makes that head's output NaN and no other's."""
    cache = Cache(27, [150, 150], 2)
    q = torch.randn((2, 4, 64), device=cuda)
    if what == "q":
        q[0, 1, 5] = float("nan")
    else:
        (cache.ks if what == "k" else cache.vs)[0][100, 1] = np.nan
        _repack(cache)
    out = ops.attention_split(q, _i32([0, 1], cuda), _i32([150, 150], cuda), 2, *cache.device(cuda))
    bad = torch.isnan(out).any(2).cpu().tolist()
    want = [[False, True, False, False], [False] * 4] if what == "q" else [[False, False, True, True], [False] * 4]
    assert bad == want
    out = ops.attention_prompt(q, _i32([0, 1, 2], cuda), _i32([0, 1], cuda), _i32([149, 149], cuda), 2,
                               *cache.device(cuda))
    assert torch.isnan(out).any(2).cpu().tolist() == want


def test_split_on_streams_and_in_a_graph(ops, cuda):
    """Another stream, a captured call replayed on new inputs and lengths, and two graphs with a workspace each."""
    cache = Cache(29, [2000, 700], 2, layers=1, layer=0)
    table, pool, page_bytes, layer = cache.device(cuda)
    q = torch.randn((2, 8, 64), device=cuda).to(torch.bfloat16)
    slot, lens = _i32([0, 1], cuda), _i32([2000, 700], cuda)
    want = ops.attention_split(q, slot, lens, 2, table, pool, page_bytes, layer)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention_split(q, slot, lens, 2, table, pool, page_bytes, layer)
    side.synchronize()
    assert torch.equal(got, want)
    need = ops.attention_split_workspace(2, 8, 2, table.shape[1])
    graphs = []
    for _ in range(2):
        out = torch.zeros_like(q)
        ws = torch.empty(need, dtype=torch.uint8, device=cuda)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.attention_split(q, slot, lens, 2, table, pool, page_bytes, layer, out=out, workspace=ws)
        graphs.append((graph, out, ws))
    for graph, out, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, _ in graphs)
    q.copy_(torch.randn_like(q))
    lens.copy_(_i32([1, 699], cuda))
    want = ops.attention_split(q, slot, lens, 2, table, pool, page_bytes, layer)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, _ in graphs)


def test_split_gives_the_same_bits_every_time(ops, cuda):
    cache = Cache(31, [5000, 3, 900], 2, layers=1, layer=0)
    q = torch.randn((3, 8, 64), device=cuda)
    args = (q, _i32([0, 1, 2], cuda), _i32([5000, 3, 900], cuda), 2, *cache.device(cuda))
    ws = torch.full((ops.attention_split_workspace(3, 8, 2, cache.max_pages),), 0xFF, dtype=torch.uint8, device=cuda)
    want = ops.attention_split(*args, workspace=ws)
    for _ in range(20):
        assert torch.equal(ops.attention_split(*args, workspace=ws), want)


# ------------------------------------------------------------------ prompts --

def _packed(lengths, prefixes):
    ends = [0]
    for n, p in zip(lengths, prefixes):
        ends.append(ends[-1] + n - p)
    return ends


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 8), (4, 1), (6, 2), (15, 3), (40, 2)])
def test_prompt_matches_64_bits(ops, cuda, kind, heads, kv_heads):
    """Packed sequences of 0 to 300 rows, some behind prefixes that end anywhere in a page."""
    lengths = [1, 64, 17, 300, 65, 129, 130, 400, 333]
    prefixes = [0, 0, 17, 0, 64, 0, 1, 271, 332]  # the third has no rows
    cache = Cache(heads * 3 + kv_heads, lengths, kv_heads)
    order = list(cache.rng.permutation(len(lengths)))
    ends = _packed([lengths[s] for s in order], [prefixes[s] for s in order])
    q, x = _queries(cache, kind, ends[-1], heads, cuda)
    for window in (0, 1, 50, 200):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = ops.attention_prompt(q, _i32(ends, cuda), _i32(order, cuda), _i32([prefixes[s] for s in order], cuda),
                                   kv_heads, *cache.device(cuda), window=window, status=status)
        assert status.item() == 0 and out.dtype == TYPES[kind]
        for i, s in enumerate(order):
            n = ends[i + 1] - ends[i]
            for r in sorted({0, 1, 2, n // 3, n // 2, n - 2, n - 1} & set(range(n))):
                _check(kind, out[ends[i] + r], cache, s, x[ends[i] + r], prefixes[s] + r, window)


@pytest.mark.parametrize("kind", list(TYPES))
def test_prompt_of_long_sequences(ops, cuda, kind):
    lengths, prefixes = [2500, 1800], [0, 1100]
    cache = Cache(41, lengths, 2, layers=1, layer=0)
    ends = _packed(lengths, prefixes)
    q, x = _queries(cache, kind, ends[-1], 8, cuda, size=3.0)
    for window in (0, 700):
        out = ops.attention_prompt(q, _i32(ends, cuda), _i32([0, 1], cuda), _i32(prefixes, cuda), 2,
                                   *cache.device(cuda), window=window)
        for s in range(2):
            n = ends[s + 1] - ends[s]
            for r in list(range(0, n, 97)) + [n - 1]:
                _check(kind, out[ends[s] + r], cache, s, x[ends[s] + r], prefixes[s] + r, window)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("window", [0, 900])
def test_prompt_whose_scores_and_scales_rise(ops, cuda, kind, window):
    """The running maximum and the common power of two of the values move all along the row."""
    cache = Cache(47, [1500], 2, layers=1, layer=0)
    cache.ks[0] = (cache.ks[0] * np.linspace(1, 10, 1500)[:, None]).astype(np.float32)
    cache.vs[0] = (cache.vs[0] * 2.0 ** (np.arange(1500) // 90)[:, None]).astype(np.float32)
    _repack(cache)
    q, x = _queries(cache, kind, 1000, 4, cuda)
    out = ops.attention_prompt(q, _i32([0, 1000], cuda), _i32([0], cuda), _i32([500], cuda), 2, *cache.device(cuda),
                               window=window)
    for r in list(range(0, 1000, 61)) + [999]:
        _check(kind, out[r], cache, 0, x[r], 500 + r, window)


def test_long_fp32_sums_do_not_drift(ops, cuda):
    """Equal weights and equal values: the result is the value.  Of the products' additions between two that round, at
    most 64 (a prompt's 8 pages of 4 products in 2 parts), each loses less than 2^-23 of what the sum then is, i/64 of
    it at the i-th: below 32 * 2^-23.  The 129 page sums and the total add up by roundings of 2^-24 of what they then
    are, 65 * 2^-24 each at most, and weights, values and the quotient round within 2^-20.  Together below 2^-16."""
    length = 8192 + 37
    cache = Cache(48, [length], 1, layers=1, layer=0)
    cache.v[0][:] = 127
    cache.vs[0][:] = np.float32(0.0123)
    _repack(cache)
    want = 127.0 * float(np.float32(0.0123))
    q = torch.zeros((40, 2, 64), device=cuda)
    out = ops.attention_prompt(q, _i32([0, 40], cuda), _i32([0], cuda), _i32([length - 40], cuda), 1, *cache.device(cuda))
    assert (out.double() / want - 1).abs().max().item() < 2.0 ** -16
    out = ops.attention_split(q[:1], _i32([0], cuda), _i32([length], cuda), 1, *cache.device(cuda))
    assert (out.double() / want - 1).abs().max().item() < 2.0 ** -16


def test_prompt_rows_agree_with_single_tokens(ops, cuda):
    """Both operators within the bound of the same rows, over every row of a chunk."""
    cache = Cache(43, [170], 2)
    q, x = _queries(cache, "f32", 100, 6, cuda)
    out = ops.attention_prompt(q, _i32([0, 100], cuda), _i32([0], cuda), _i32([70], cuda), 2, *cache.device(cuda))
    one = ops.attention_split(q, _i32([0] * 100, cuda), _i32(range(71, 171), cuda), 2, *cache.device(cuda))
    for r in range(100):
        _check("f32", out[r], cache, 0, x[r], 70 + r, 0)
        _check("f32", one[r], cache, 0, x[r], 70 + r, 0)


@pytest.mark.parametrize("kind", list(TYPES))
def test_prompt_leaves_other_rows_alone(ops, cuda, kind):
    """Rows before the first sequence and behind the last keep what they held, strided outputs keep their gaps."""
    cache = Cache(45, [40, 90], 2)
    q, x = _queries(cache, kind, 160, 4, cuda)
    wide = torch.full((160, 512), 3.0, device=cuda, dtype=TYPES[kind])
    out = wide[:, 64:320].unflatten(1, (4, 64))
    ops.attention_prompt(q, _i32([7, 47, 137], cuda), _i32([0, 1], cuda), _i32([0, 0], cuda), 2, *cache.device(cuda),
                         out=out)
    assert torch.all(wide[:7] == 3.0) and torch.all(wide[137:] == 3.0)
    assert torch.all(wide[:, :64] == 3.0) and torch.all(wide[:, 320:] == 3.0)
    for r in (7, 46, 47, 100, 136):
        s = int(r >= 47)
        _check(kind, out[r], cache, s, x[r], r - (47 if s else 7), 0)


def test_prompt_bad_sequences(ops, cuda):
    """Bad slots, positions and pages make that sequence's rows NaN with status 2, the others' are done; a
    sequence whose offsets descend or leave the rows is skipped with status 2."""
    lengths = [100, 200, 64, 70]
    cache = Cache(47, lengths, 2)
    cache.table[1, 2] = cache.num_pages + 1
    q = torch.randn((400, 4, 64), device=cuda).half()
    ends = [0, 100, 300, 310, 320, 330, 400]
    slots, starts = [0, 1, 9, 2, 2, 3], [0, 0, 0, -1, 64 * cache.max_pages - 5, 0]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = ops.attention_prompt(q, _i32(ends, cuda), _i32(slots, cuda), _i32(starts, cuda), 2, *cache.device(cuda),
                               status=status)
    assert status.item() == 2
    x = q.double().cpu().numpy()
    for r in (0, 50, 99):
        _check("f16", out[r], cache, 0, x[r], r, 0)
    for r in (330, 350, 399):
        _check("f16", out[r], cache, 3, x[r], r - 330, 0)
    assert torch.isnan(out[228:330]).all()  # from the missing page's first position on, and the bad sequences
    for bad, done in (([0, 50, 30], range(50)), ([0, 70, 500], range(70)), ([-3, 40, 90], range(40, 90))):
        status.zero_()
        out = torch.full_like(q, 9.0)
        ops.attention_prompt(q, _i32(bad, cuda), _i32([0, 3], cuda), _i32([0, 0], cuda), 2, *cache.device(cuda),
                             out=out, status=status)
        assert status.item() == 2
        for r in (done[0], done[-1]):
            _check("f16", out[r], cache, 3 if done[0] else 0, x[r], r - done[0], 0)
        rest = torch.ones(400, dtype=torch.bool)
        rest[list(done)] = False
        assert torch.all(out[rest.to(cuda)] == 9.0)


def test_prompt_on_streams_and_in_a_graph(ops, cuda):
    cache = Cache(49, [300, 80], 2, layers=1, layer=0)
    table, pool, page_bytes, layer = cache.device(cuda)
    q = torch.randn((380, 4, 64), device=cuda).to(torch.bfloat16)
    ends, slot, start = _i32([0, 300, 380], cuda), _i32([0, 1], cuda), _i32([0, 0], cuda)
    call = lambda out=None: ops.attention_prompt(q, ends, slot, start, 2, table, pool, page_bytes, layer, out=out)
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(out)
    q.copy_(torch.randn_like(q))
    ends.copy_(_i32([0, 33, 113], cuda))
    out.fill_(9.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:113], call()[:113])
    assert torch.all(out[113:] == 9.0)


def test_attention_wrapper_refusals(ops, cuda):
    cache = Cache(51, [10], 2)
    pages = cache.device(cuda)
    q, one = torch.zeros((1, 4, 64), device=cuda), _i32([1], cuda)
    with pytest.raises(ValueError):
        ops.attention_split(q[..., :32], one, one, 2, *pages)
    with pytest.raises(TypeError):
        ops.attention_split(q, one, one, 2, *pages, out=q.half())
    with pytest.raises(ValueError):
        ops.attention_split(q, one, one, 2, *pages, out=torch.zeros((2, 4, 64), device=cuda))
    with pytest.raises(ValueError):
        ops.attention_prompt(q, one, one, one, 2, *pages)
    with pytest.raises(Exception, match="query heads"):
        ops.attention_split(torch.zeros((1, 5, 64), device=cuda), one, one, 2, *pages)


@pytest.mark.parametrize("kind", list(TYPES))
def test_outputs_in_the_queries_place(ops, cuda, kind):
    """out may be q: rows inside a warp, over a CTA's warps and over CTAs, and a prompt of several tiles."""
    cache = Cache(61, [9000, 700, 65, 3], 2)
    lengths = cache.lengths
    q, _ = _queries(cache, kind, 4, 8, cuda)
    args = (_i32(range(4), cuda), _i32(lengths, cuda), 2, *cache.device(cuda))
    want = ops.attention_split(q, *args)
    assert ops.attention_split(q, *args, out=q) is q
    assert torch.equal(q, want)
    q, _ = _queries(cache, kind, 1000, 8, cuda)
    args = (_i32([0, 700, 990, 1000], cuda), _i32([1, 0, 2], cuda), _i32([0, 8000, 55], cuda), 2, *cache.device(cuda))
    want = ops.attention_prompt(q, *args)
    assert ops.attention_prompt(q, *args, out=q) is q
    assert torch.equal(q, want)


def test_windows_of_any_size(ops, cuda):
    """A window longer than the sequence is none, up to the largest int."""
    cache = Cache(62, [1500, 3], 2)
    q, _ = _queries(cache, "bf16", 600, 4, cuda)
    args = (_i32([0, 597, 600], cuda), _i32([0, 1], cuda), _i32([903, 0], cuda), 2, *cache.device(cuda))
    single = (_i32([0, 1], cuda), _i32([1500, 3], cuda), 2, *cache.device(cuda))
    want, want_split = ops.attention_prompt(q, *args), ops.attention_split(q[:2], *single)
    for window in (1500, 1 << 20, 2 ** 31 - 1):
        assert torch.equal(ops.attention_prompt(q, *args, window=window), want)
        assert torch.equal(ops.attention_split(q[:2], *single, window=window), want_split)


def test_two_calls_at_once(ops, cuda):
    """The same rows on two streams, each with its own workspace and pages of one pool."""
    cache = Cache(63, [4000, 300, 3000, 64], 2)
    table, pool, page_bytes, layer = cache.device(cuda)
    q, _ = _queries(cache, "f16", 4, 8, cuda)
    slots, lengths = _i32(range(4), cuda), _i32(cache.lengths, cuda)
    want = ops.attention_split(q, slots, lengths, 2, table, pool, page_bytes, layer)
    prompt = (_i32([0, 4], cuda), _i32([2], cuda), _i32([2996], cuda), 2, table, pool, page_bytes, layer)
    want_prompt = ops.attention_prompt(q, *prompt)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append((ops.attention_split(q, slots, lengths, 2, table, pool, page_bytes, layer),
                            ops.attention_prompt(q, *prompt)))
    torch.cuda.synchronize()
    for split, prompted in got:
        assert torch.equal(split, want) and torch.equal(prompted, want_prompt)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_a_device_that_is_not_current(ops, cuda):
    """The tensors' device decides, whichever is current; its kernels' attributes are set there too."""
    cache = Cache(64, [700, 90], 2)
    other = torch.device("cuda", 1)
    results = []
    for device in (cuda, other):
        q = torch.from_numpy(np.random.default_rng(5).normal(size=(2, 8, 64))).float().to(device)
        pages = cache.device(device)
        slots = torch.tensor([0, 1], dtype=torch.int32, device=device)
        lengths = torch.tensor([700, 90], dtype=torch.int32, device=device)
        results.append([ops.attention_split(q, slots, lengths, 2, *pages),
                        ops.attention_prompt(q, torch.tensor([0, 1, 2], dtype=torch.int32, device=device), slots,
                                             lengths - 1, 2, *pages), *ops.kv_gather(slots, lengths - 1, 2, *pages),
                        ops.logits_process(q.flatten(1))])
    for a, b in zip(*results):
        assert b.device == other and torch.equal(a.cpu(), b.cpu())



# ----------------------------------------------------------------- together --

def test_a_request_from_prompt_to_token(ops, cuda):
    """Two requests: their rows into empty pages, the prompt's attention, a token step, the logits' penalties and the
    pick; the cache's own kernel (ndl_attention_paged) reads the same pages."""
    from paged_support import processed

    cache = Cache(53, [0, 0], 2, layers=2, layer=1, spare_pages=8, spare_columns=3)
    cache.table[0, :3], cache.table[1, :3] = [4, 1, 7], [2, 0, 5]
    table, pool, page_bytes, layer = cache.device(cuda)
    lens = [130, 64]
    rows = sum(lens)
    qkv = torch.randn((rows, 4 * 64 + 4 * 64), device=cuda)
    part = lambda t, a, b: t[:, a:b].unflatten(1, ((b - a) // 64, 64))
    slot = _i32([0] * 130 + [1] * 64, cuda)
    pos = _i32(list(range(130)) + list(range(64)), cuda)
    pages = (table, pool, page_bytes, layer)
    ops.kv_append(part(qkv, 256, 384), part(qkv, 384, 512), slot, pos, *pages)
    out = ops.attention_prompt(part(qkv, 0, 256), _i32([0, 130, 194], cuda), _i32([0, 1], cuda), _i32([0, 0], cuda), 2,
                               *pages)
    new = torch.randn((2, 512), device=cuda)
    ops.kv_append(part(new, 256, 384), part(new, 384, 512), _i32([0, 1], cuda), _i32(lens, cuda), *pages)
    token = ops.attention_split(part(new, 0, 256), _i32([0, 1], cuda), _i32([131, 65], cuda), 2, *pages)
    k, v = ops.kv_gather(slot, pos, 2, *pages)
    nk, nv = ops.kv_gather(_i32([0, 1], cuda), _i32(lens, cuda), 2, *pages)
    from paged_support import bound as limit_of
    for s in range(2):
        at = slice(0, 130) if s == 0 else slice(130, 194)
        keys = torch.cat([k[at], nk[s:s + 1]]).double().cpu().numpy()
        values = torch.cat([v[at], nv[s:s + 1]]).double().cpu().numpy()
        q = part(qkv, 0, 256)[at].double().cpu().numpy()
        checks = [(out[at][r], q[r], r) for r in (0, 63, lens[s] - 1)]
        checks.append((token[s], part(new, 0, 256)[s].double().cpu().numpy(), lens[s]))
        for got, x, p in checks:
            want, size, reach = attend(x, keys, values, p)
            limit = limit_of("f32", want, size, reach, p + 1, np.abs(values).max())
            assert np.all(np.abs(got.double().cpu().numpy() - want) <= limit)
    # the engine's decode kernel on the same pages (its own query quantizer makes it coarser: a step of 1/127 a dim)
    from attention_support import K_ORDER
    head_q = part(new, 0, 256)[:, ::2].contiguous()
    q8, qs = ops.quantize_rows(head_q.reshape(4, 64))
    paged = torch.empty_like(q8)
    paged[:, torch.from_numpy(K_ORDER).to(cuda)] = q8
    old = ops.attention_paged(paged.view(2, 2, 64), qs.view(2, 2), _i32([0, 1], cuda), _i32(lens, cuda), *pages)
    mine = ops.attention_split(head_q, _i32([0, 1], cuda), _i32([131, 65], cuda), 2, *pages)
    exact_q = (q8.float() * qs[:, None]).view(2, 2, 64)
    same = ops.attention_split(exact_q, _i32([0, 1], cuda), _i32([131, 65], cuda), 2, *pages)
    for s in range(2):
        at = slice(0, 130) if s == 0 else slice(130, 194)
        keys = torch.cat([k[at], nk[s:s + 1]]).double().cpu().numpy()
        values = torch.cat([v[at], nv[s:s + 1]]).double().cpu().numpy()
        want, size, reach = attend(exact_q[s].double().cpu().numpy(), keys, values, lens[s])
        limit = limit_of("f32", want, size, reach, lens[s] + 1, np.abs(values).max())
        assert np.all(np.abs((same[s] - old[s]).double().cpu().numpy()) <= 2 * limit)
    assert mine.shape == same.shape
    w = torch.randn((256, 500), device=cuda)
    logits = token.flatten(1) @ w
    history = [[3, 3, 499, 7], [1]]
    got = ops.logits_process(logits, tokens=_i32(sum(history, []), cuda), token_offsets=_i32([0, 4, 5], cuda),
                             prompt_lens=_i32([1, 0], cuda), repetition=torch.tensor([1.3, 2.0], device=cuda),
                             presence=torch.tensor([0.5, 0.1], device=cuda))
    x = logits.cpu().numpy()
    want = np.stack([processed(x[0], history[0], 1, 1.3, None, 0.5), processed(x[1], history[1], 0, 2.0, None, 0.1)])
    assert np.array_equal(got.cpu().numpy(), want)
    assert got.argmax(1).tolist() == want.argmax(1).tolist()
