"""Penalties, biases and masks on logits (ndl_logits_process): every step is
one IEEE operation, so the results equal the definition bit for bit."""
import numpy as np
import pytest
import torch

from paged_support import processed

pytestmark = pytest.mark.gpu


def _i32(a, cuda):
    return torch.tensor(np.asarray(a, dtype=np.int64), dtype=torch.int32, device=cuda)


def _f32(a, cuda):
    return torch.tensor(np.asarray(a), dtype=torch.float32, device=cuda)


def _case(seed, rows, vocab, most_tokens, most_bias, words=None):
    rng = np.random.default_rng(seed)
    x = (4 * rng.normal(size=(rows, vocab))).astype(np.float32)
    x[rng.random(x.shape) < 0.02] = 0.0
    # a few ids often, some outside the vocabulary
    tokens = [list((vocab * rng.random(int(rng.integers(0, most_tokens + 1))) ** 3).astype(int)) for _ in range(rows)]
    for t in tokens:
        if len(t) > 3:
            t[1], t[2] = -1, vocab + 5
    bias = [[(int(rng.integers(-1, vocab + 2)), float(np.float32(rng.normal()))) for _ in range(rng.integers(0, most_bias + 1))]
            for _ in range(rows)]
    words = (vocab + 31) // 32 if words is None else words
    return dict(x=x, tokens=tokens, prompt=[int(rng.integers(0, len(t) + 2)) for t in tokens],
                repetition=rng.uniform(0.7, 1.6, rows).astype(np.float32),
                frequency=rng.uniform(-0.5, 1, rows).astype(np.float32),
                presence=rng.uniform(-0.5, 1, rows).astype(np.float32), bias=bias,
                mask=rng.integers(0, 1 << 32, (rows, words), dtype=np.uint32))


def _offsets(lists):
    return np.concatenate([[0], np.cumsum([len(t) for t in lists])])


def _run(ops, cuda, c, logits=None, mask_index=None, **kw):
    flat = [t for row in c["tokens"] for t in row]
    pairs = [b for row in c["bias"] for b in row]
    return ops.logits_process(
        torch.from_numpy(c["x"]).to(cuda) if logits is None else logits, tokens=_i32(flat, cuda),
        token_offsets=_i32(_offsets(c["tokens"]), cuda), prompt_lens=_i32(c["prompt"], cuda),
        repetition=_f32(c["repetition"], cuda), frequency=_f32(c["frequency"], cuda),
        presence=_f32(c["presence"], cuda), bias_ids=_i32([i for i, _ in pairs], cuda),
        bias_values=_f32([b for _, b in pairs], cuda), bias_offsets=_i32(_offsets(c["bias"]), cuda),
        mask=torch.from_numpy(c["mask"].view(np.int32)).to(cuda),
        mask_index=None if mask_index is None else _i32(mask_index, cuda), **kw)


def _want(c, mask_index=None):
    rows = []
    for r in range(len(c["x"])):
        m = r if mask_index is None else mask_index[r]
        rows.append(processed(c["x"][r], c["tokens"][r], c["prompt"][r], c["repetition"][r], c["frequency"][r],
                              c["presence"][r], c["bias"][r], c["mask"][m] if m >= 0 else None))
    return np.stack(rows)


@pytest.mark.parametrize("rows,vocab,tokens,bias", [(1, 1, 3, 1), (3, 31, 50, 4), (2, 4096, 300, 9), (4, 4097, 900, 40),
                                                    (5, 8192, 2000, 100), (2, 51865, 500, 30), (7, 333, 0, 0),
                                                    (21, 51865, 400, 60), (40, 30001, 6000, 900)])
def test_logits_match_the_definition(ops, cuda, rows, vocab, tokens, bias):
    c = _case(rows + vocab, rows, vocab, tokens, bias)
    assert np.array_equal(_run(ops, cuda, c).cpu().numpy(), _want(c))
    index = [(r * 5 + 1) % rows if r % 3 else -1 for r in range(rows)]
    assert np.array_equal(_run(ops, cuda, c, mask_index=index).cpu().numpy(), _want(c, index))


def test_short_masks_and_empty_ones(ops, cuda):
    """Ids past the mask's words are disallowed; a mask that allows nothing leaves a row of -inf."""
    c = _case(5, 3, 700, 50, 5, words=4)
    c["mask"][1] = 0
    got = _run(ops, cuda, c).cpu().numpy()
    assert np.array_equal(got, _want(c))
    assert np.all(np.isneginf(got[1])) and np.all(np.isneginf(got[:, 128:]))


def test_special_values(ops, cuda):
    """Infinities and NaN: masked places become -inf whatever they held, the others follow the arithmetic."""
    c = _case(6, 2, 200, 100, 10)
    c["x"][:, ::9] = np.inf
    c["x"][:, 1::9] = -np.inf
    c["x"][:, 2::9] = np.nan
    c["x"][:, 3::9] = np.finfo(np.float32).max
    c["x"][:, 4::9] = np.finfo(np.float32).min
    with np.errstate(all="ignore"):
        want = _want(c)
    got = _run(ops, cuda, c).cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)


def test_each_part_alone_and_none(ops, cuda):
    c = _case(7, 4, 5000, 400, 20)
    x = torch.from_numpy(c["x"]).to(cuda)
    assert torch.equal(ops.logits_process(x), x)
    tok = dict(tokens=_i32([t for r in c["tokens"] for t in r], cuda), token_offsets=_i32(_offsets(c["tokens"]), cuda))
    assert torch.equal(ops.logits_process(x, **tok), x)
    for name in ("repetition", "frequency", "presence"):
        got = ops.logits_process(x, **tok, **{name: _f32(c[name], cuda)})
        want = np.stack([processed(c["x"][r], c["tokens"][r], 0, **{name: c[name][r]}) for r in range(4)])
        assert np.array_equal(got.cpu().numpy(), want), name
    got = ops.logits_process(x, mask=torch.from_numpy(c["mask"].view(np.int32)).to(cuda))
    assert np.array_equal(got.cpu().numpy(), np.stack([processed(c["x"][r], mask=c["mask"][r]) for r in range(4)]))
    got = ops.logits_process(x, bias_ids=_i32([5, 5, 9], cuda), bias_values=_f32([1, 2, 3], cuda),
                             bias_offsets=_i32([0, 0, 3, 3, 3], cuda))
    want = x.clone()
    want[1, 5] += 2
    want[1, 9] += 3
    assert torch.equal(got, want)


def test_large_calls_in_place_and_unaligned(ops, cuda):
    """The two-kernel form: in place, rows that lie differently to 16 bytes in and out, and a captured call."""
    c = _case(12, 12, 90001, 300, 40)
    want = _want(c)
    wide = torch.full((12, 90007), 2.5, device=cuda)
    wide[:, 2:90003] = torch.from_numpy(c["x"]).to(cuda)
    out = torch.full((12, 90010), 1.5, device=cuda)
    _run(ops, cuda, c, logits=wide[:, 2:90003], out=out[:, 1:90002])
    assert np.array_equal(out[:, 1:90002].cpu().numpy(), want)
    assert torch.all(out[:, :1] == 1.5) and torch.all(out[:, 90002:] == 1.5)
    x = torch.from_numpy(c["x"]).to(cuda)
    _run(ops, cuda, c, logits=x, out=x)
    assert np.array_equal(x.cpu().numpy(), want)
    x.copy_(torch.from_numpy(c["x"]))
    mask = torch.from_numpy(c["mask"].view(np.int32)).to(cuda)
    tok = dict(tokens=_i32([t for r in c["tokens"] for t in r], cuda), token_offsets=_i32(_offsets(c["tokens"]), cuda),
               repetition=_f32(c["repetition"], cuda), mask=mask)
    want = ops.logits_process(x, **tok)
    y = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.logits_process(x, out=y, **tok)
    for _ in range(2):
        y.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_in_place_strided_and_unaligned_rows(ops, cuda):
    """In place, with row strides no vector load divides, and from an odd start."""
    c = _case(8, 3, 1001, 200, 10)
    want = _want(c)
    x = torch.from_numpy(c["x"]).to(cuda)
    assert _run(ops, cuda, c, logits=x, out=x) is x
    assert np.array_equal(x.cpu().numpy(), want)
    wide = torch.full((3, 1031), 2.5, device=cuda)
    wide[:, 13:1014] = torch.from_numpy(c["x"]).to(cuda)
    out = torch.full((3, 1040), 1.5, device=cuda)
    _run(ops, cuda, c, logits=wide[:, 13:1014], out=out[:, 4:1005])
    assert np.array_equal(out[:, 4:1005].cpu().numpy(), want)
    assert torch.all(out[:, :4] == 1.5) and torch.all(out[:, 1005:] == 1.5)
    assert torch.all(wide[:, :13] == 2.5) and torch.all(wide[:, 1014:] == 2.5)


@pytest.mark.parametrize("rows,vocab", [(3, 300), (150, 8190)])
def test_bad_mask_rows(ops, cuda, rows, vocab):
    """A mask row past the last gives a NaN row with status 2, in the small form and the large one."""
    if rows > 3:
        x = torch.randn((rows, vocab), device=cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        mask = torch.full((2, 256), -1, dtype=torch.int32, device=cuda)
        got = ops.logits_process(x, tokens=_i32([1, 2], cuda), token_offsets=_i32([0] * 8 + [2] * (rows - 7), cuda),
                                 presence=torch.ones(rows, device=cuda), mask=mask, mask_index=_i32([0] * 7 + [2] + [1] * (rows - 8), cuda),
                                 status=status)
        assert status.item() == 2 and torch.isnan(got[7]).all()
        assert torch.equal(got[:7], x[:7]) and torch.equal(got[8:], x[8:])
        return
    c = _case(9, 3, 300, 20, 2)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = _run(ops, cuda, c, mask_index=[2, 3, -4], status=status)
    assert status.item() == 2
    assert torch.isnan(got[1]).all()
    want = _want(c, [2, 0, -1])
    assert np.array_equal(got[[0, 2]].cpu().numpy(), want[[0, 2]])


def test_long_histories_and_a_graph(ops, cuda):
    """One id many thousands of times, and a captured call replayed with grown lists."""
    vocab = 9000
    c = _case(10, 2, vocab, 0, 0)
    c["tokens"] = [[77] * 20000 + [8999] * 3, list(range(vocab))]
    c["prompt"] = [5, vocab - 1]
    assert np.array_equal(_run(ops, cuda, c).cpu().numpy(), _want(c))
    x = torch.randn((2, vocab), device=cuda)
    tokens, offsets = torch.zeros(64, dtype=torch.int32, device=cuda), _i32([0, 0, 0], cuda)
    pen = _f32([1.5, 0.5], cuda)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.logits_process(x, out=out, tokens=tokens, token_offsets=offsets, repetition=pen, presence=pen)
    for n in (0, 3, 30):
        ids = [(7 * i) % vocab for i in range(2 * n)]
        tokens[:2 * n] = _i32(ids, cuda)
        offsets.copy_(_i32([0, n, 2 * n], cuda))
        graph.replay()
        torch.cuda.synchronize()
        y = x.cpu().numpy()
        want = np.stack([processed(y[r], ids[r * n:(r + 1) * n], 0, pen[r].item(), None, pen[r].item())
                         for r in range(2)])
        assert np.array_equal(out.cpu().numpy(), want)


def test_before_the_engines_sampler(ops, pkg, cuda):
    """The engine's own logits of a step, adjusted on its stream and picked: a strong repetition penalty changes a
    loop, a bias decides."""
    from needle_cs_b200.engine import BatchedEngine, SyntheticDecoder

    model = SyntheticDecoder(layers=1, dim=128, heads=2, head_dim=64, ffn=256, vocab=1000, seed=3)
    with BatchedEngine(model, slots=2, context_length=64, chunk_size=8) as eng:
        eng.forward_batch([5, 9], [0, 1], [0, 1])
        ids = eng.sample_argmax()
        rows = np.stack([eng.batch_logits_row(r) for r in range(2)])
        assert ids.tolist() == rows.argmax(1).tolist()
        got = ops.logits_process(torch.from_numpy(rows).to(cuda), bias_ids=_i32([int(ids[0]), 17], cuda),
                                 bias_values=_f32([-1e4, 1e4], cuda), bias_offsets=_i32([0, 1, 2], cuda))
        want = np.stack([processed(rows[0], bias=[(int(ids[0]), -1e4)]), processed(rows[1], bias=[(17, 1e4)])])
        assert np.array_equal(got.cpu().numpy(), want)
        assert got.argmax(1).tolist()[1] == 17 and got.argmax(1).tolist()[0] != ids[0]


def test_many_ids_in_place_unaligned_and_in_a_graph(ops, cuda):
    """Calls of millions of ids: in place, rows that lie differently to 16 bytes in and out, one row with lists too
    long for shared memory, one whose mask does not exist, and a captured call."""
    rows, vocab = 40, 90001
    c = _case(16, rows, vocab, 300, 40)
    c["tokens"][3] = [(i * i) % (vocab + 7) for i in range(9000)]
    c["prompt"][3] = 4000
    c["bias"][3] = [((31 * i) % vocab, float(np.float32(0.01 * i))) for i in range(500)]
    want = _want(c)
    x = torch.from_numpy(c["x"]).to(cuda)
    wide = torch.full((rows, vocab + 6), 2.5, device=cuda)
    wide[:, 2:vocab + 2] = x
    out = torch.full((rows, vocab + 9), 1.5, device=cuda)
    _run(ops, cuda, c, logits=wide[:, 2:vocab + 2], out=out[:, 1:vocab + 1])
    assert np.array_equal(out[:, 1:vocab + 1].cpu().numpy(), want)
    assert torch.all(out[:, :1] == 1.5) and torch.all(out[:, vocab + 1:] == 1.5)
    y = x.clone()
    _run(ops, cuda, c, logits=y, out=y)
    assert np.array_equal(y.cpu().numpy(), want)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    index = list(range(rows))
    index[7] = rows
    got = _run(ops, cuda, c, mask_index=index, status=status)
    assert status.item() == 2 and torch.isnan(got[7]).all()
    keep = [r for r in range(rows) if r != 7]
    assert np.array_equal(got[keep].cpu().numpy(), want[keep])
    mask = torch.from_numpy(c["mask"].view(np.int32)).to(cuda)
    tok = dict(tokens=_i32([t for r in c["tokens"] for t in r], cuda), token_offsets=_i32(_offsets(c["tokens"]), cuda),
               repetition=_f32(c["repetition"], cuda), mask=mask)
    eager = ops.logits_process(x, **tok)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.logits_process(x, out=y, **tok)
    for _ in range(2):
        y.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_large_calls_whose_lists_are_empty(ops, cuda):
    """What follows on the stream reads the whole result, although no row's list has work."""
    rows, vocab = 128, 1 << 15
    x = torch.randn((rows, vocab), device=cuda)
    zero = torch.zeros(rows + 1, dtype=torch.int32, device=cuda)
    some = _i32([1, 2, 3], cuda)
    mask = torch.full((rows, vocab // 32), 0x0F0F0F0F, dtype=torch.int32, device=cuda)
    allowed = (torch.arange(vocab, device=cuda) & 4) == 0
    want = torch.where(allowed, x, torch.full_like(x, -torch.inf))
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    for _ in range(20):
        out.zero_()
        ops.logits_process(x, out=out, tokens=some, token_offsets=zero, repetition=torch.ones(rows, device=cuda), mask=mask)
        copy = out.clone()
        assert torch.equal(copy, want)
