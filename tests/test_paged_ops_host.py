"""Refusals of the row, attention and logits operators: every one is decided
on the host before any device work, so none needs a GPU.  The addresses are
aligned numbers that nothing reads."""
import ctypes

import pytest

OK, INVALID = 0, 100
P = 4096  # stands for a device address
BLOCK = 8704


def _append(**kw):
    a = dict(k=P, ks=128, v=P, vs=128, type=0, slot=P, pos=P, rows=3, kv=2, table=P, slots=2, pages=4, pool=P,
             bytes=2 * 2 * BLOCK, num=8, layer=1, status=None, stream=None)
    a.update(kw)
    return "ndl_kv_append", list(a.values())


def _gather(**kw):
    a = dict(slot=P, pos=P, rows=3, kv=2, table=P, slots=2, pages=4, pool=P, bytes=2 * 2 * BLOCK, num=8, layer=1, k=P,
             ks=128, v=P, vs=128, type=0, status=None, stream=None)
    a.update(kw)
    return "ndl_kv_gather", list(a.values())


def _prompt(**kw):
    a = dict(q=P, qs=256, type=0, seq_rows=P, seq_slot=P, seq_pos=P, sequences=2, rows=3, heads=4, kv=2, scale=0.125,
             window=0, table=P, slots=2, pages=4, pool=P, bytes=2 * 2 * BLOCK, num=8, layer=1, out=P, os=256,
             status=None, stream=None)
    a.update(kw)
    return "ndl_attention_prompt", list(a.values())


def _split(**kw):
    a = dict(q=P, qs=256, type=0, slot=P, len=P, rows=3, heads=4, kv=2, scale=0.125, window=0, table=P, slots=2,
             pages=4, pool=P, bytes=2 * 2 * BLOCK, num=8, layer=1, out=P, os=256, ws=P, wsb=1 << 30, status=None,
             stream=None)
    a.update(kw)
    return "ndl_attention_split", list(a.values())


def _logits(**kw):
    a = dict(x=P, ldx=100, y=P, ldy=100, rows=2, vocab=100, tokens=P, n_tokens=5, token_offsets=P, prompt=P, rep=P,
             freq=P, pres=P, bias_ids=P, bias_values=P, n_bias=3, bias_offsets=P, mask=P, mask_rows=2, words=4,
             mask_index=P, status=None, stream=None)
    a.update(kw)
    return "ndl_logits_process", list(a.values())


CACHE = [dict(kv=0), dict(slots=0), dict(pages=0), dict(num=0), dict(layer=-1), dict(layer=2), dict(table=None),
         dict(pool=None), dict(pool=P + 8), dict(bytes=2 * 2 * BLOCK - 16), dict(bytes=2 * 2 * BLOCK + 8),
         dict(pages=1 << 26), dict(rows=-1), dict(type=3), dict(type=-1), dict(table=P + 2)]
ROWS = CACHE + [dict(k=None), dict(v=None), dict(slot=None), dict(pos=None), dict(ks=127), dict(ks=130), dict(vs=64),
                dict(k=P + 4), dict(v=P + 8), dict(type=1, ks=132), dict(rows=1 << 30, kv=2)]
ATTENTION = CACHE + [dict(q=None), dict(out=None), dict(heads=3), dict(heads=0), dict(scale=0.0),
                     dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-1.0), dict(window=-1),
                     dict(qs=255), dict(os=128), dict(q=P + 2), dict(out=P + 4), dict(rows=1 << 30)]


@pytest.mark.parametrize("make,bad", [(_append, ROWS), (_gather, ROWS),
                                      (_prompt, ATTENTION + [dict(sequences=-1), dict(seq_rows=None),
                                                             dict(seq_slot=None), dict(seq_pos=None)]),
                                      (_split, ATTENTION + [dict(slot=None), dict(len=None), dict(ws=P + 4)]),
                                      (_logits, [dict(rows=-1), dict(vocab=0), dict(x=None), dict(y=None),
                                                 dict(ldx=99), dict(ldy=99), dict(ldy=104), dict(tokens=None),
                                                 dict(token_offsets=None), dict(bias_ids=None),
                                                 dict(bias_values=None), dict(bias_offsets=None),
                                                 dict(n_tokens=-1), dict(n_bias=-1), dict(words=0),
                                                 dict(mask_rows=0), dict(mask_rows=1, mask_index=None),
                                                 dict(mask=None), dict(rows=70000)])],
                         ids=["append", "gather", "prompt", "split", "logits"])
def test_refusals(pkg, make, bad):
    lib = pkg.lib()
    for kw in bad:
        name, args = make(**kw)
        assert getattr(lib, name)(*args) == INVALID, (name, kw)
        assert lib.ndl_last_error(), (name, kw)


@pytest.mark.parametrize("make", [_append, _gather, _prompt, _split, _logits],
                         ids=["append", "gather", "prompt", "split", "logits"])
def test_no_rows_is_no_work(pkg, make):
    """A call without rows succeeds without a launch, so it does here without a GPU too."""
    name, args = make(rows=0)
    assert getattr(pkg.lib(), name)(*args) == OK


def test_no_sequences_is_no_work(pkg):
    name, args = _prompt(sequences=0, seq_slot=None, seq_pos=None)
    assert getattr(pkg.lib(), name)(*args) == OK


def test_split_workspace(pkg):
    """The workspace is what the call asks for: a byte less is refused."""
    size = pkg.lib().ndl_attention_split_workspace
    assert size(0, 8, 8, 16) == 0 and size(4, 0, 8, 16) == 0 and size(4, 8, 0, 16) == 0 and size(4, 8, 8, 0) == 0
    assert size(4, 9, 8, 16) == 0  # heads that kv_heads does not divide: no such call
    for rows, heads, kv, pages in [(1, 8, 8, 2000), (3, 4, 2, 4), (64, 32, 8, 128)]:
        need = size(rows, heads, kv, pages)
        if need:
            name, args = _split(rows=rows, heads=heads, kv=kv, pages=pages, qs=heads * 64, os=heads * 64,
                                bytes=2 * kv * BLOCK, wsb=need - 1)
            assert getattr(pkg.lib(), name)(*args) == INVALID
            assert str(need) in pkg.lib().ndl_last_error().decode()
            name, args = _split(rows=rows, heads=heads, kv=kv, pages=pages, qs=heads * 64, os=heads * 64,
                                bytes=2 * kv * BLOCK, ws=None)
            assert getattr(pkg.lib(), name)(*args) == INVALID


def test_wrappers_refuse_host_tensors(ops):
    """The Python entry points check their tensors before the library sees an address."""
    import torch

    table, pool = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(BLOCK, dtype=torch.uint8)
    x, one = torch.zeros((1, 1, 64)), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.kv_append(x, x, one, one, table, pool, BLOCK, 0)
    with pytest.raises(TypeError):
        ops.kv_gather(one, one, 1, table, pool, BLOCK, 0)
    with pytest.raises(TypeError):
        ops.attention_prompt(x, torch.zeros(2, dtype=torch.int32), one, one, 1, table, pool, BLOCK, 0)
    with pytest.raises(TypeError):
        ops.attention_split(x, one, one, 1, table, pool, BLOCK, 0)
    with pytest.raises(TypeError):
        ops.attention_split(x.double(), one, one, 1, table, pool, BLOCK, 0)
    with pytest.raises(TypeError):
        ops.logits_process(torch.zeros((1, 8)))


def test_plain_implementation_of_the_logits():
    """The test oracle itself, by hand."""
    import numpy as np
    from paged_support import processed

    x = np.array([2.0, -2.0, 0.5, 1.0, 3.0], np.float32)
    got = processed(x, tokens=[0, 1, 1, 3, 99, -1], prompt=1, repetition=2.0, frequency=0.25, presence=0.125,
                    bias=[(4, 1.0), (4, -1.0), (2, 0.5)], mask=[0b01111])
    assert np.array_equal(got, np.array([1.0, -4.0 - 0.5 - 0.125, 1.0, 0.5 - 0.25 - 0.125, -np.inf], np.float32))
