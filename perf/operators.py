"""Cases of the operators that serve a request over the paged int8 KV cache: the whole-prompt attention, the
single-token attention split over the cache's length, the cache's write and read of rows, and the logits'
penalties, biases and masks.

Every attention and cache case works on a pool of pages in the library's layout (64 positions a page, int8 keys
and values with one fp32 scale per (position, head), 64-dim heads), its pages in random order, as a page
allocator leaves them.  Lengths are drawn from the case's own `lens` number, inputs from the seed.

`run` gives the operators' plain form, or with `own` the library's calls.
"""
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
PAGE, DIM, RECORD = 64, 64, 8704
MASKED = 0.3  # share of the rows that carry a grammar mask


def listed():
    return [
        # the first prompt of an idle server: one short request, its latency is the time to the first token
        dict(name="prompt: one of 37 rows, fp32", op="prompt", type="f32", heads=8, kv_heads=8, layers=2, seqs=1,
             rows_lo=37, rows_hi=37, prefix_lo=0, prefix_hi=0, window=0, lens=1),
        # one step of the continuous-batching trace's arrivals: many prompts of U[32,384] tokens in the engine's fp32
        dict(name="prompt: 32 arrivals, fp32", op="prompt", type="f32", heads=8, kv_heads=8, layers=2, seqs=32,
             rows_lo=32, rows_hi=384, prefix_lo=0, prefix_hi=0, window=0, lens=2),
        # prompt chunks behind shared prefixes on a sliding-window layer, six query heads to a kv head
        dict(name="prompt: chunks, window, fp16", op="prompt", type="f16", heads=12, kv_heads=2, layers=1, seqs=24,
             rows_lo=1, rows_hi=256, prefix_lo=0, prefix_hi=4096, window=1024, lens=3),
        # one long document: the compute-bound end
        dict(name="prompt: one of 8192, bf16", op="prompt", type="bf16", heads=32, kv_heads=8, layers=1, seqs=1,
             rows_lo=8192, rows_hi=8192, prefix_lo=0, prefix_hi=0, window=0, lens=4),
        # one session's next token: latency
        dict(name="token: one session, fp32", op="token", type="f32", heads=8, kv_heads=8, layers=2, seqs=1,
             rows_lo=1000, rows_hi=1000, window=0, lens=5),
        # a 64-session decode step, caches of U[16,512]
        dict(name="token: 64 sessions, fp32", op="token", type="f32", heads=8, kv_heads=8, layers=2, seqs=64,
             rows_lo=16, rows_hi=512, window=0, lens=6),
        # one session behind a very long context: one row has to fill the card
        dict(name="token: one at 100003, bf16", op="token", type="bf16", heads=32, kv_heads=8, layers=1, seqs=1,
             rows_lo=100003, rows_hi=100003, window=0, lens=7),
        # a full decode batch with contexts of very different lengths: bandwidth
        dict(name="token: 256 to 8192, bf16", op="token", type="bf16", heads=32, kv_heads=8, layers=1, seqs=256,
             rows_lo=64, rows_hi=8192, window=0, lens=8),
        # the cache rows of one decode step of 64 sessions
        dict(name="cache: 64 rows, fp32", op="cache", type="f32", kv_heads=8, layers=2, seqs=64, rows_lo=16,
             rows_hi=512, count=64, lens=9),
        # the cache rows of a few long prompts
        dict(name="cache: 16384 rows, bf16", op="cache", type="bf16", kv_heads=8, layers=1, seqs=7, rows_lo=1024,
             rows_hi=8192, count=16384, lens=10),
        # the next token of one tool call
        dict(name="logits: one row", op="logits", rows=1, vocab=8192, hist_lo=300, hist_hi=300, bias_hi=8, lens=11),
        # a batch over a speech model's vocabulary
        dict(name="logits: 256 rows of 51865", op="logits", rows=256, vocab=51865, hist_lo=0, hist_hi=1024,
             bias_hi=64, lens=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    while True:  # until it costs no more than the largest listed case, and its padded scores fit beside it
        case = _drawn(rng)
        w = work(case)
        rows = case["rows_hi"] if case["op"] == "prompt" else 0
        if w["flops"] <= 2.7e11 and w["bytes"] <= 1.09e9 and (
                not rows or case["seqs"] * case["heads"] * rows * (rows + case["prefix_hi"]) <= 1 << 31):
            return case


def _drawn(rng):
    op = rng.choice(["prompt", "prompt", "token", "token", "cache", "logits"])
    lens = rng.randrange(1 << 30)
    if op == "logits":
        rows, vocab = _log(rng, 1, 256), _log(rng, 300, 51865)
        hi = _log(rng, 1, 2048)
        return dict(op=op, rows=rows, vocab=vocab, hist_lo=0, hist_hi=hi, bias_hi=_log(rng, 1, 256), lens=lens)
    type_ = rng.choice(["f32", "f16", "bf16"])
    kv = rng.choice([1, 2, 3, 4, 8])
    if op == "cache":
        count, seqs = _log(rng, 1, 16384), _log(rng, 1, 64)
        longest = max(-(-count // seqs), _log(rng, 64, 8192))
        return dict(op=op, type=type_, kv_heads=kv, layers=rng.choice([1, 2]), seqs=seqs, rows_lo=longest,
                    rows_hi=longest, count=count, lens=lens)
    group = rng.choice([1, 2, 3, 4, 6, 8, 12])
    heads = kv * group
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    if op == "token":
        seqs = _log(rng, 1, 256)
        hi = _log(rng, 1, min(100003, (1 << 20) // seqs))
        return dict(op=op, type=type_, heads=heads, kv_heads=kv, layers=rng.choice([1, 2]), seqs=seqs,
                    rows_lo=rng.choice([0, 1, hi]), rows_hi=hi, window=window, lens=lens)
    seqs = _log(rng, 1, 64)
    hi = _log(rng, 1, 8192 // max(1, round(seqs ** 0.5)))
    prefix = rng.choice([0, 0, _log(rng, 1, 4096)])
    return dict(op=op, type=type_, heads=heads, kv_heads=kv, layers=rng.choice([1, 2]), seqs=seqs,
                rows_lo=rng.choice([0, 1, hi]), rows_hi=hi, prefix_lo=0, prefix_hi=prefix, window=window, lens=lens)


def _lengths(case):
    """(rows, prefix) of each sequence of an attention or cache case."""
    r = random.Random(case["lens"])
    rows = [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    if case["op"] == "prompt" and sum(rows) == 0:
        rows[0] = 1
    prefix = [r.randint(case.get("prefix_lo", 0), case.get("prefix_hi", 0)) for _ in range(case["seqs"])]
    return rows, prefix


def _attended(case):
    """Pairs (query, position) and cached positions read at least once, over all sequences of an attention case."""
    rows, prefix = _lengths(case)
    w = case["window"]
    if case["op"] == "token":
        n = sum(min(x, w) if w else x for x in rows)
        return n, n
    pairs = read = 0
    for n, p in zip(rows, prefix):
        if not n:
            continue
        first = max(0, p - w + 1) if w else 0
        read += p + n - first
        if w:
            short = max(0, min(n, w - p))  # the first rows see every position up to their own
            pairs += short * p + short * (short + 1) // 2 + (n - short) * w
        else:
            pairs += n * p + n * (n + 1) // 2
    return pairs, read


def _history(case):
    r = random.Random(case["lens"])
    total = [r.randint(case["hist_lo"], case["hist_hi"]) for _ in range(case["rows"])]
    prompt = [r.randint(0, n) for n in total]
    bias = [r.randint(0, case["bias_hi"]) for _ in total]
    masked = [i if r.random() < MASKED else -1 for i in range(case["rows"])]
    return total, prompt, bias, masked


def work(case):
    if case["op"] == "logits":
        total, _, bias, masked = _history(case)
        cells = case["rows"] * case["vocab"]
        words = sum(m >= 0 for m in masked) * -(-case["vocab"] // 32)
        return {"bytes": 8 * cells + 4 * sum(total) + 8 * sum(bias) + 4 * words, "flops": 2 * sum(total)}
    e = SIZES[case["type"]]
    if case["op"] == "cache":
        vectors = 2 * case["count"] * case["kv_heads"]  # a key and a value of 64 for each (row, head)
        return {"bytes": vectors * (2 * DIM * e + 2 * (DIM + 4)), "flops": vectors * 4 * DIM}
    pairs, read = _attended(case)
    q = case["seqs"] if case["op"] == "token" else sum(_lengths(case)[0])
    return {"bytes": read * case["kv_heads"] * 2 * (DIM + 4) + 2 * q * case["heads"] * DIM * e,
            "flops": 4 * DIM * case["heads"] * pairs}


# ------------------------------------------------------------------ inputs --

def _maps(device):
    """Byte of (position, dim) of a record's keys and values, and of each position's two scales."""
    p, d = torch.arange(PAGE, device=device)[:, None], torch.arange(DIM, device=device)[None, :]
    key = ((p >> 4) * 1024 + (d >> 5) * 512 + ((p & 7) * 4 + ((d >> 2) & 3)) * 16
           + (((p >> 3) & 1) + 2 * ((d >> 4) & 1)) * 4 + (d & 3))
    value = 4608 + d * 64 + ((((p >> 4) ^ ((d >> 1) & 3)) << 4) | (p & 15))
    p = p[:, 0]
    return {"key": key, "value": value, "key_scale": 1024 + 2 * ((p & 7) * 4 + ((p >> 4) & 3)) + ((p >> 3) & 1),
            "value_scale": 1088 + p}


def _codes(x):
    peak = x.abs().amax(-1)
    scale = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
    return (x * (1 / scale)[..., None]).round().clamp(-128, 127).to(torch.int8), scale


def _pool(case, lengths, gen, maps):
    """A filled pool, its page table and the geometry: pages in random order, unused table entries -1."""
    need = [-(-n // PAGE) for n in lengths]
    total, widest = max(1, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    counts = torch.tensor(need, device="cuda")
    col = torch.arange(widest, device="cuda")
    at = (starts[:, None] + col).clamp(max=total - 1)
    table = torch.where(col < counts[:, None], order[at], torch.full_like(order[at], -1)).contiguous()
    layers, kv = case["layers"], case["kv_heads"]
    pool = torch.zeros((total, layers, kv, RECORD), dtype=torch.uint8, device="cuda")
    rec = pool[:, layers - 1]
    for at, scale_at in (("key", "key_scale"), ("value", "value_scale")):
        codes, scale = _codes(torch.randn((total, kv, PAGE, DIM), generator=gen, device="cuda"))
        rec[..., maps[at].reshape(-1)] = codes.reshape(total, kv, -1).view(torch.uint8)
        rec.view(torch.float32)[..., maps[scale_at]] = scale
        del codes, scale
    return pool.reshape(-1), table


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, gen)
    maps = _maps("cuda")
    rows, prefix = _lengths(case)
    pool, table = _pool(case, [a + b for a, b in zip(rows, prefix)], gen, maps)
    kv, layers, dtype = case["kv_heads"], case["layers"], TYPES[case["type"]]
    state = dict(case=case, pool=pool, table=table, maps=maps, page_bytes=layers * kv * RECORD, layer=layers - 1)
    if case["op"] == "cache":
        # the sessions' last positions, shared out evenly, session by session
        r = random.Random(case["lens"] + 1)
        left, slots, places = case["count"], [], []
        for s, n in enumerate(rows):
            take = min(n, -(-left // (len(rows) - s)))
            slots += [s] * take
            places += range(n - take, n)
            left -= take
        spare = [(s, p) for s, n in enumerate(rows) for p in range(n)] if left else []
        spare = list(set(spare) - set(zip(slots, places)))
        spare.sort()
        for s, p in r.sample(spare, min(left, len(spare))):
            slots.append(s)
            places.append(p)
        state |= {x: torch.randn((len(slots), kv, DIM), generator=gen, device="cuda").to(dtype) for x in ("k", "v")}
        return state | dict(row_slot=_i32(slots), row_pos=_i32(places))
    count = sum(rows) if case["op"] == "prompt" else len(rows)
    # scores of standard deviation 2 over the row: some positions matter, many still add up
    state["q"] = (2 * torch.randn((count, case["heads"], DIM), generator=gen, device="cuda")).to(dtype)
    slots = list(range(len(rows)))
    random.Random(case["lens"] + 1).shuffle(slots)  # row i serves slot slots[i]
    if case["op"] == "token":
        return state | dict(row_slot=_i32(slots), row_len=_i32([rows[s] for s in slots]))
    ends = [0]
    for s in slots:
        ends.append(ends[-1] + rows[s])
    # the longest prompt and the most positions, which the plain form pads to
    state["longest"], state["widest"] = max(rows), max(a + b for a, b in zip(rows, prefix))
    return state | dict(seq_rows=_i32(ends), seq_slot=_i32(slots), seq_pos=_i32([prefix[s] for s in slots]))


def _prepare_logits(case, gen):
    total, prompt, bias, masked = _history(case)
    rows, vocab = case["rows"], case["vocab"]
    offsets = [0]
    bias_offsets = [0]
    for n, b in zip(total, bias):
        offsets.append(offsets[-1] + n)
        bias_offsets.append(bias_offsets[-1] + b)

    def rand(n, lo, hi):
        return lo + (hi - lo) * torch.rand(n, generator=gen, device="cuda")

    # text repeats itself: small ids far more often than large ones
    ids = (vocab * rand(offsets[-1], 0, 1) ** 3).to(torch.int32).clamp(max=vocab - 1)
    bias_ids = torch.randint(0, vocab, (bias_offsets[-1],), generator=gen, device="cuda", dtype=torch.int32)
    words = -(-vocab // 32)
    mask = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=gen, device="cuda").to(torch.int32)
    mask &= torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=gen, device="cuda").to(torch.int32)
    return dict(case=case, logits=4 * torch.randn((rows, vocab), generator=gen, device="cuda"), tokens=ids,
                token_offsets=_i32(offsets), prompt_lens=_i32(prompt), repetition=rand(rows, 1.0, 1.5),
                frequency=rand(rows, 0.0, 0.5), presence=rand(rows, 0.0, 0.5), bias_ids=bias_ids,
                bias_values=rand(bias_offsets[-1], -5, 5), bias_offsets=_i32(bias_offsets), mask=mask,
                mask_index=_i32(masked))


# -------------------------------------------------------------- plain forms --

def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return {"prompt": _plain_prompt, "token": _plain_token, "cache": _plain_cache, "logits": _plain_logits}[op](state)


def _plain_records(state, slots):
    """Keys and values [slots, kv heads, positions, 64] in 32 bits of the listed slots' whole page lists."""
    kv, maps = state["case"]["kv_heads"], state["maps"]
    rec = state["pool"].view(-1, state["case"]["layers"], kv, RECORD)
    rec = rec[state["table"][slots].clamp(min=0).long(), state["layer"]]  # [slots, pages, kv, RECORD]
    scales = rec.view(torch.float32)

    def part(at, scale_at):
        codes = rec[..., maps[at].reshape(-1)].view(torch.int8).unflatten(-1, (PAGE, DIM)).float()
        codes.mul_(scales[..., maps[scale_at]][..., None])
        return codes.transpose(1, 2).flatten(2, 3)

    return part("key", "key_scale"), part("value", "value_scale")


def _plain_softmax(scores, seen, values):
    scores.masked_fill_(~seen, float("-inf"))
    peak = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(peak == float("-inf"), torch.zeros_like(peak), peak)).exp_()
    total = scores.sum(-1, keepdim=True)
    return (scores @ values) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_token(state):
    case, q = state["case"], state["q"]
    keys, values = _plain_records(state, state["row_slot"].long())
    kv = case["kv_heads"]
    place = torch.arange(keys.shape[2], device="cuda")
    length = state["row_len"].long()[:, None, None, None]
    seen = place < length
    if case["window"]:
        seen = seen & (place >= length - case["window"])
    scores = (q.float() * 0.125).unflatten(1, (kv, -1)) @ keys.transpose(2, 3)
    return _plain_softmax(scores, seen, values).flatten(1, 2).to(q.dtype)


def _plain_prompt(state):
    case, q = state["case"], state["q"]
    kv, group, longest = case["kv_heads"], case["heads"] // case["kv_heads"], state["longest"]
    keys, values = _plain_records(state, state["seq_slot"].long())
    keys, values = keys[:, :, :state["widest"]], values[:, :, :state["widest"]]
    start = state["seq_rows"].long()
    line = torch.arange(longest, device="cuda")
    at = start[:-1, None] + line  # [sequences, longest]: the packed row, where it exists
    there = line < (start[1:] - start[:-1])[:, None]
    padded = (q.float() * 0.125)[at.clamp(max=q.shape[0] - 1)]  # [sequences, longest, heads, 64]
    padded = padded.unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [s, kv, group * longest, 64]
    place = torch.arange(keys.shape[2], device="cuda")
    row_pos = (state["seq_pos"].long()[:, None] + line).repeat(1, group)[:, None, :, None]
    seen = place <= row_pos
    if case["window"]:
        seen = seen & (place > row_pos - case["window"])
    out = _plain_softmax(padded @ keys.transpose(2, 3), seen, values)
    out = out.unflatten(2, (group, longest)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[there].to(q.dtype)


def _plain_cache(state):
    case, maps = state["case"], state["maps"]
    rec = state["pool"].view(-1, case["layers"], case["kv_heads"], RECORD)
    place = state["row_pos"].long()
    page = state["table"][state["row_slot"].long(), place // PAGE].long()
    place = place % PAGE
    got = []
    for x, at, scale_at in ((state["k"], "key", "key_scale"), (state["v"], "value", "value_scale")):
        codes, scale = _codes(x.float())
        head = torch.arange(case["kv_heads"], device="cuda")
        where = (page[:, None], state["layer"], head)
        rec[where[0][..., None], state["layer"], head[:, None], maps[at][place][:, None]] = codes.view(torch.uint8)
        rec.view(torch.float32)[where + (maps[scale_at][place][:, None],)] = scale
        back = rec[where[0][..., None], state["layer"], head[:, None], maps[at][place][:, None]].view(torch.int8)
        back = back.float() * rec.view(torch.float32)[where + (maps[scale_at][place][:, None],)][..., None]
        got.append(back.to(x.dtype))
    return got


def _plain_logits(state):
    x = state["logits"].clone()
    rows, vocab = x.shape
    ids, start = state["tokens"].long(), state["token_offsets"].long()
    entry = torch.arange(ids.numel(), device="cuda")
    row = torch.bucketize(entry, start[1:], right=True)
    output = entry - start[row] >= state["prompt_lens"].long()[row]
    cell = row * vocab + ids
    ever = torch.zeros(rows * vocab, device="cuda").scatter_(0, cell, 1.0).view(rows, vocab) > 0
    times = torch.zeros(rows * vocab, device="cuda").scatter_add_(0, cell, output.float()).view(rows, vocab)
    r = state["repetition"][:, None]
    x = torch.where(ever, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(times > 0, x - state["frequency"][:, None] * times, x)
    x = torch.where(times > 0, x - state["presence"][:, None], x)
    # of a row's biases for one id the last counts
    start = state["bias_offsets"].long()
    entry = torch.arange(state["bias_ids"].numel(), device="cuda")
    cell = torch.bucketize(entry, start[1:], right=True) * vocab + state["bias_ids"].long()
    last = torch.full((rows * vocab,), -1, device="cuda").scatter_reduce_(0, cell, entry, "amax").view(rows, vocab)
    bias = torch.cat([state["bias_values"], torch.zeros(1, device="cuda")])[last]
    x = torch.where(last >= 0, x + bias, x)
    bit = torch.arange(vocab, device="cuda")
    mask = state["mask"][state["mask_index"].long().clamp(min=0)]
    allowed = (mask[:, bit >> 5] >> (bit & 31)) & 1 > 0
    return x.masked_fill(~allowed & (state["mask_index"] >= 0)[:, None], float("-inf"))


# ------------------------------------------------------- the library's calls --

def _ops():
    import __graft_entry__

    __graft_entry__.load_package()
    import needle_cs_b200.ops

    return needle_cs_b200.ops


def _run_own(state):
    ops, case = _ops(), state["case"]
    if case["op"] == "logits":
        return ops.logits_process(
            state["logits"], tokens=state["tokens"], token_offsets=state["token_offsets"],
            prompt_lens=state["prompt_lens"], repetition=state["repetition"], frequency=state["frequency"],
            presence=state["presence"], bias_ids=state["bias_ids"], bias_values=state["bias_values"],
            bias_offsets=state["bias_offsets"], mask=state["mask"], mask_index=state["mask_index"])
    pages = (state["table"], state["pool"], state["page_bytes"], state["layer"])
    if case["op"] == "cache":
        ops.kv_append(state["k"], state["v"], state["row_slot"], state["row_pos"], *pages)
        return list(ops.kv_gather(state["row_slot"], state["row_pos"], case["kv_heads"], *pages,
                                  dtype=state["k"].dtype))
    if case["op"] == "token":
        return ops.attention_split(state["q"], state["row_slot"], state["row_len"], case["kv_heads"], *pages,
                                   window=case["window"])
    return ops.attention_prompt(state["q"], state["seq_rows"], state["seq_slot"], state["seq_pos"],
                                case["kv_heads"], *pages, window=case["window"])


# ------------------------------------------------------------------- exact --

def _exact_slot(state, pages, first, last):
    """Keys and values [kv heads, positions first..last, 64] in 64 bits: each code's byte from the layout's formulas
    (keys in 16-byte groups of two rows' four dims twice, values dim by dim)."""
    kv, layers = state["case"]["kv_heads"], state["case"]["layers"]
    raw = state["pool"].view(-1, layers * kv, RECORD)
    place = torch.arange(first, last, device="cuda")
    page, p = pages[place // 64].long(), place % 64
    head = state["layer"] * kv + torch.arange(kv, device="cuda")
    d = torch.arange(64, device="cuda")
    lane = (p % 8)[:, None] * 4 + (d // 4) % 4
    register = (p // 8 % 2)[:, None] + (d // 16 % 2) * 2
    key_at = (p // 16)[:, None] * 1024 + (d // 32) * 512 + lane * 16 + register * 4 + d % 4
    value_at = 4608 + d * 64 + ((p // 16)[:, None] ^ (d // 2 % 4)) * 16 + (p % 16)[:, None]
    score_lane = (p % 8) * 4 + p // 16
    key_scale_at, value_scale_at = 4096 + 8 * score_lane + 4 * (p // 8 % 2), 4352 + 4 * p
    byte = torch.arange(4, device="cuda")

    def part(at, scale_at):
        codes = raw[page[:, None], head[:, None, None], at].view(torch.int8).double()
        scales = raw[page[:, None], head[:, None, None], (scale_at[:, None] + byte)]
        return codes * scales.contiguous().view(torch.float32).double()

    return part(key_at, key_scale_at), part(value_at, value_scale_at)


def _exact_attention(q, keys, values, first, row_pos, window):
    """[rows, heads, 64] of rows at `row_pos` over positions first.. of one sequence."""
    rows, heads, _ = q.shape
    group = heads // keys.shape[0]
    scores = torch.einsum("rkgd,kpd->kgrp", q.double().view(rows, -1, group, 64), keys) / 8
    place = first + torch.arange(keys.shape[1], device="cuda")
    bad = place > row_pos[:, None]
    if window:
        bad = bad | (place + window <= row_pos[:, None])
    scores.masked_fill_(bad, float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1)
    return (torch.einsum("kgrp,kpd->kgrd", scores, values) / total[..., None]).permute(2, 0, 1, 3).reshape(rows, heads, 64)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(state)
    if case["op"] == "cache":
        return [_exact_code(state[x].double()) for x in ("k", "v")]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    w = case["window"]
    if case["op"] == "token":
        for i, (s, n) in enumerate(zip(state["row_slot"].tolist(), state["row_len"].tolist())):
            if n:
                first = max(0, n - w) if w else 0
                k, v = _exact_slot(state, state["table"][s], first, n)
                out[i:i + 1] = _exact_attention(state["q"][i:i + 1], k, v, first, _i32([n - 1]), w)
        return out
    ends = state["seq_rows"].tolist()
    for i, (s, p) in enumerate(zip(state["seq_slot"].tolist(), state["seq_pos"].tolist())):
        n = ends[i + 1] - ends[i]
        for a in range(0, n, 2048):
            b = min(n, a + 2048)
            first = max(0, p + a - w + 1) if w else 0
            k, v = _exact_slot(state, state["table"][s], first, p + b)
            at = p + torch.arange(a, b, device="cuda")
            out[ends[i] + a:ends[i] + b] = _exact_attention(state["q"][ends[i] + a:ends[i] + b], k, v, first, at, w)
    return out


def _exact_code(x):
    """The cache's quantizer is defined with its three roundings to 32 bits (the stored scale, its inverse, the
    product), which decide the code next to a border: they are kept, all else is in 64 bits."""
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    scale[scale == 0] = 1
    return torch.round((x * (1 / scale).float().double()).float().double()) * scale


def _exact_logits(state):
    out = state["logits"].double()
    vocab = out.shape[1]
    ends, bias_ends = state["token_offsets"].tolist(), state["bias_offsets"].tolist()
    for i, (n, m) in enumerate(zip(state["prompt_lens"].tolist(), state["mask_index"].tolist())):
        x, ids = out[i], state["tokens"][ends[i]:ends[i + 1]].long()
        r, f, p = (state[a][i].double() for a in ("repetition", "frequency", "presence"))
        seen = torch.bincount(ids, minlength=vocab) > 0
        times = torch.bincount(ids[n:], minlength=vocab)
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x) - f * times - p * (times > 0)
        given = dict(zip(state["bias_ids"][bias_ends[i]:bias_ends[i + 1]].tolist(),
                         state["bias_values"][bias_ends[i]:bias_ends[i + 1]].tolist()))
        if given:
            x[list(given)] += torch.tensor(list(given.values()), dtype=torch.float64, device="cuda")
        if m >= 0:
            bits = (state["mask"][m].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.reshape(-1)[:vocab] == 0] = float("-inf")
        out[i] = x
    return out
