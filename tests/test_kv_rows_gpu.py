"""Rows of keys and values into the pages and back (ndl_kv_append,
ndl_kv_gather): codes and scales equal the quantizer's definition bit for
bit, and nothing else in the pool changes."""
import numpy as np
import pytest
import torch

from paged_support import TYPES, Cache, quantized, records

pytestmark = pytest.mark.gpu


def _places(cache, rng, count):
    """`count` distinct (slot, position) pairs in random order."""
    every = [(s, p) for s, n in enumerate(cache.lengths) for p in range(n)]
    pick = rng.permutation(len(every))[:count]
    return [every[i] for i in pick]


def _i32(a, cuda):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=cuda)


def _expected(cache, places, k, v):
    """The pool's bytes after the rows, from a copy of the bytes before."""
    from attention_support import K_BYTE, K_OFF, KS_OFF, S_SLOT, V_BYTE, V_OFF, VS_OFF

    pool = cache.pool.copy()
    kc, ksc = quantized(k)
    vc, vsc = quantized(v)
    for r, (s, p) in enumerate(places):
        for h in range(cache.kv_heads):
            rec = pool[cache.table[s, p // 64], cache.layer, h]
            j = p % 64
            rec[K_OFF + K_BYTE[j]] = kc[r, h].view(np.uint8)
            rec[V_OFF + V_BYTE[j]] = vc[r, h].view(np.uint8)
            rec[KS_OFF:KS_OFF + 256].view(np.float32)[S_SLOT[j]] = ksc[r, h]
            rec[VS_OFF:VS_OFF + 256].view(np.float32)[j] = vsc[r, h]
    return pool


def _rows(cache, kind, count, rng, cuda):
    """Values with zeros, a zero vector, ties and a wide range."""
    x = rng.normal(size=(2, count, cache.kv_heads, 64)) * 2.0 ** rng.integers(-20, 12, (2, count, cache.kv_heads, 1))
    x[rng.random(x.shape) < 0.05] = 0.0
    if count > 2:
        x[:, 1] = 0.0
        x[:, 2] = np.round(x[:, 2] * 4) / 4
        x[:, 2, :, 0] = 127.0
    t = torch.from_numpy(x).to(TYPES[kind])
    return t[0].to(cuda), t[1].to(cuda), t.float().numpy()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("order", ["random", "runs"])
def test_append_writes_exactly_its_rows(ops, cuda, kind, order):
    cache = Cache(3, [200, 1, 64, 130, 0, 17], 3)
    rng = np.random.default_rng(4)
    if order == "random":
        places = _places(cache, rng, 150)
    else:  # whole prompts and chunks, at starts that are no multiples of anything
        places = ([(0, p) for p in range(5, 200)] + [(1, 0)] + [(2, p) for p in range(64)]
                  + [(3, p) for p in range(16, 113)] + [(5, 16)])
    k, v, x = _rows(cache, kind, len(places), rng, cuda)
    table, pool, page_bytes, layer = cache.device(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slot, pos = zip(*places)
    ops.kv_append(k, v, _i32(slot, cuda), _i32(pos, cuda), table, pool, page_bytes, layer, status=status)
    assert status.item() == 0
    assert np.array_equal(pool.cpu().numpy(), _expected(cache, places, x[0], x[1]).reshape(-1))


def test_append_equals_the_row_quantizer(ops, cuda):
    cache = Cache(5, [70], 2)
    x = torch.randn((70, 2, 64), device=cuda)
    table, pool, page_bytes, layer = cache.device(cuda)
    ops.kv_append(x, x, _i32([0] * 70, cuda), _i32(range(70), cuda), table, pool, page_bytes, layer)
    q, s = ops.quantize_rows(x.reshape(140, 64))
    kc, vc, ks, vs = records(pool.cpu().numpy(), cache)
    pages = cache.table[0, :2]
    for got, scale in ((kc, ks), (vc, vs)):
        at = got[pages].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:70]
        assert np.array_equal(at, q.cpu().numpy().reshape(70, 2, 64))
        assert np.array_equal(scale[pages].transpose(0, 2, 1).reshape(-1, 2)[:70], s.cpu().numpy().reshape(70, 2))


@pytest.mark.parametrize("kind", list(TYPES))
def test_gather_returns_the_stored_values(ops, cuda, kind):
    cache = Cache(6, [100, 0, 64, 1], 3)
    rng = np.random.default_rng(7)
    places = _places(cache, rng, 90)
    slot, pos = zip(*places)
    k, v = ops.kv_gather(_i32(slot, cuda), _i32(pos, cuda), 3, *cache.device(cuda), dtype=TYPES[kind])
    for got, codes, scales in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        want = np.stack([codes[s][p].astype(np.float32) * scales[s][p][:, None] for s, p in places])
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(TYPES[kind]))


def test_strided_rows_of_a_fused_projection(ops, cuda):
    """k and v as columns of one [rows, q | k | v] matrix, and gather into such columns."""
    cache = Cache(8, [65, 20], 2)
    rng = np.random.default_rng(9)
    places = _places(cache, rng, 33)
    slot, pos = (_i32(a, cuda) for a in zip(*places))
    qkv = torch.randn((33, 4 * 64 + 2 * 2 * 64), device=cuda)
    k, v = qkv[:, 256:384].unflatten(1, (2, 64)), qkv[:, 384:].unflatten(1, (2, 64))
    table, pool, page_bytes, layer = cache.device(cuda)
    ops.kv_append(k, v, slot, pos, table, pool, page_bytes, layer)
    want = _expected(cache, places, k.cpu().numpy(), v.cpu().numpy())
    assert np.array_equal(pool.cpu().numpy(), want.reshape(-1))
    out = torch.full((33, 512), 7.0, device=cuda)
    ops.kv_gather(slot, pos, 2, table, pool, page_bytes, layer, k=out[:, 128:256].unflatten(1, (2, 64)),
                  v=out[:, 384:].unflatten(1, (2, 64)))
    k2, v2 = ops.kv_gather(slot, pos, 2, table, pool, page_bytes, layer)
    assert torch.equal(out[:, 128:256], k2.flatten(1)) and torch.equal(out[:, 384:], v2.flatten(1))
    assert torch.all(out[:, :128] == 7.0) and torch.all(out[:, 256:384] == 7.0)


def test_padding_and_bad_rows(ops, cuda):
    """Padding rows write nothing and gather zeros, bad ones set the status and gather NaN, the rest are done."""
    cache = Cache(10, [64, 30], 2)
    cache.table[1, 1] = cache.num_pages + 3  # a page outside the pool
    slot = [0, 0, -1, 2, 1, 1, 1, 0]
    pos = [-1, 5, 3, 3, 70, 64 * cache.max_pages, 7, -5]
    good = [(1, (0, 5)), (6, (1, 7))]
    k = torch.randn((8, 2, 64), device=cuda)
    v = torch.randn((8, 2, 64), device=cuda)
    table, pool, page_bytes, layer = cache.device(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.kv_append(k, v, _i32(slot, cuda), _i32(pos, cuda), table, pool, page_bytes, layer, status=status)
    assert status.item() == 2
    rows = [r for r, _ in good]
    want = _expected(cache, [p for _, p in good], k.cpu().numpy()[rows], v.cpu().numpy()[rows])
    assert np.array_equal(pool.cpu().numpy(), want.reshape(-1))
    status.zero_()
    gk, gv = ops.kv_gather(_i32(slot, cuda), _i32(pos, cuda), 2, table, pool, page_bytes, layer, status=status)
    assert status.item() == 2
    for x in (gk, gv):
        assert torch.all(x[[0, 7]] == 0) and torch.all(torch.isnan(x[[2, 3, 4, 5]])) and not torch.any(torch.isnan(x[rows]))
    status.zero_()
    ops.kv_append(k[:1], v[:1], _i32([0], cuda), _i32([-1], cuda), table, pool, page_bytes, layer, status=status)
    assert status.item() == 0


def test_wrapper_refusals(ops, cuda):
    cache = Cache(11, [10], 2)
    table, pool, page_bytes, layer = cache.device(cuda)
    k, one = torch.zeros((1, 2, 64), device=cuda), _i32([0], cuda)
    with pytest.raises(TypeError):
        ops.kv_append(k, k.half(), one, one, table, pool, page_bytes, layer)
    with pytest.raises(ValueError):
        ops.kv_append(k, k[:, :1], one, one, table, pool, page_bytes, layer)
    with pytest.raises(ValueError):
        ops.kv_append(k.transpose(1, 2).contiguous().transpose(1, 2), k, one, one, table, pool, page_bytes, layer)
    with pytest.raises(ValueError):
        ops.kv_append(k, k, _i32([0, 0], cuda), one, table, pool, page_bytes, layer)
    with pytest.raises(TypeError):
        ops.kv_append(k, k, one.long(), one, table, pool, page_bytes, layer)


def test_many_rows_of_runs_singles_and_padding(ops, cuda):
    """Enough rows for the larger blocks: chunks at any start, single tokens and padding, shuffled, so runs cross
    blocks and chunks of pages; nothing else in the pool changes, and the rows come back."""
    cache = Cache(21, [130] * 60, 3)
    rng = np.random.default_rng(22)
    pieces = []
    for s in rng.permutation(60):  # each slot in pieces of 1 to 45 positions, some positions left out
        at = int(rng.integers(0, 9))
        while at < 130:
            n = int(rng.integers(1, 46)) if rng.random() < 0.7 else 1
            pieces.append([(s, p) for p in range(at, min(130, at + n))])
            at += n + int(rng.integers(0, 3))
    places = []
    for i in rng.permutation(len(pieces)):
        places += pieces[i]
        places += [(int(rng.integers(-1, 60)), -1)] * int(rng.integers(0, 3) // 2)
    rows = len(places)
    assert (rows + 31) // 32 * 3 >= 296
    k, v, x = _rows(cache, "bf16", rows, rng, cuda)
    table, pool, page_bytes, layer = cache.device(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slot, pos = (_i32(a, cuda) for a in zip(*places))
    ops.kv_append(k, v, slot, pos, table, pool, page_bytes, layer, status=status)
    real = [r for r, (_, p) in enumerate(places) if p >= 0]
    want = _expected(cache, [places[r] for r in real], x[0][real], x[1][real])
    assert np.array_equal(pool.cpu().numpy(), want.reshape(-1))
    for kind in TYPES:
        got = ops.kv_gather(slot, pos, 3, table, pool, page_bytes, layer, dtype=TYPES[kind], status=status)
        for g, r in zip(got, x):
            codes, scales = quantized(r)
            back = torch.from_numpy(codes.astype(np.float32) * scales[..., None]).to(TYPES[kind])
            back[[p < 0 for _, p in places]] = 0
            assert torch.equal(g.cpu(), back)
    assert status.item() == 0


def test_append_and_gather_on_a_stream_and_in_a_graph(ops, cuda):
    """Captured on a side stream and replayed with other rows and places."""
    cache = Cache(23, [100, 90], 2)
    rng = np.random.default_rng(24)
    table, pool, page_bytes, layer = cache.device(cuda)
    k, v = torch.zeros((40, 2, 64), device=cuda), torch.zeros((40, 2, 64), device=cuda)
    slot, pos = _i32([0] * 40, cuda), _i32([-1] * 40, cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.kv_append(k, v, slot, pos, table, pool, page_bytes, layer)
        back = ops.kv_gather(slot, pos, 2, table, pool, page_bytes, layer)
    for _ in range(3):
        places = _places(cache, rng, 25) + [(0, -1)] * 15
        x = rng.normal(size=(2, 40, 2, 64)).astype(np.float32)
        for t, value in ((k, x[0]), (v, x[1]), (slot, [s for s, _ in places]), (pos, [p for _, p in places])):
            t.copy_(torch.as_tensor(np.asarray(value)))
        graph.replay()
        for got, value in zip(back, x):
            codes, scales = quantized(value)
            want = codes.astype(np.float32) * scales[..., None]
            want[25:] = 0
            assert np.array_equal(got.cpu().numpy(), want)
