"""Cases, plain forms and 64-bit forms of three serving operators: appending to
an 8-bit paged K/V cache, attention over that cache, and sampling rows of
logits.  A case is a dict of plain values whose "op" says which operator it
runs; `own` chooses between the plain form and the library's entry points."""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _library():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qora-tts-12hz-1.7b_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import qtts_b200
    return qtts_b200


# ---- cases ---------------------------------------------------------------------


def _append(name, seqs, rows, start, heads, kv_heads, hd, dtype, norm, pad=0):
    return {"name": name, "op": "append", "seqs": seqs, "rows": rows, "start": start, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "norm": norm, "pad": pad}


def _attend(name, seqs, rows, length, window, heads, kv_heads, hd, dtype, pad=0):
    return {"name": name, "op": "attend", "seqs": seqs, "rows": rows, "length": length, "window": window,
            "heads": heads, "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "pad": pad}


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p, spread):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "spread": spread}


def listed():
    return [
        # one utterance's next token: the smallest append, all latency
        _append("append one token", 1, 1, 300, 16, 8, 128, "f32", True),
        # a decode step of a full wave of utterances, with some slots idle
        _append("append 512 tokens", 512, 1, 2000, 16, 8, 128, "f32", True, pad=7),
        # chunks of prompts that continue caches ending inside a page
        _append("append prompt chunks", 16, 611, 900, 16, 8, 128, "bf16", True, pad=33),
        # one utterance decoding over a cache of a few seconds of speech
        _attend("attend one token", 1, 1, 265, 0, 16, 8, 128, "f32"),
        # 64 utterances with ragged prompts, one frame each
        _attend("attend 64 tokens", 64, 1, 530, 0, 16, 8, 128, "f32", pad=3),
        # one token over a cache near the position table's end: few rows, a long axis
        _attend("attend long cache", 1, 1, 32003, 0, 16, 8, 128, "f16"),
        # a large serving batch over long caches
        _attend("attend 256 long caches", 256, 1, 4099, 0, 16, 8, 128, "bf16"),
        # a prompt's prefill in 16 bits: four chunks of 1000 rows over caches to 3001 positions
        _attend("attend prompt chunks", 4, 1000, 3001, 0, 16, 8, 128, "bf16", pad=5),
        # the speech decoder's layer shape: 16 heads of 64, window 72, every frame of an utterance
        _attend("attend windowed frames", 1, 500, 500, 72, 16, 16, 64, "f32"),
        # the code predictor's heads for a wave of utterances
        _sample("sample 256 codes", 256, 2048, "f32", 50, 1.0, 0.0, 3.0),
        # one row over the text vocabulary, nucleus sampling
        _sample("sample one text row", 1, 151936, "f32", 0, 0.95, 0.0, 3.0),
        # a batch over the text vocabulary with every filter on
        _sample("sample 128 text rows", 128, 151936, "bf16", 1000, 0.95, 0.02, 2.5),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (16, 16), (4, 2), (2, 1), (16, 4), (8, 1), (16, 1), (12, 4)])
    hd = rng.choice([64, 128, 128])
    pad = rng.choice([0, 0, 1, 5, 40])
    if op == "append":
        rows = _log(rng, 1, 1500)
        c = _append("", _log(rng, 1, max(1, min(600, 9776 // rows))), rows, rng.choice([0, _log(rng, 1, 3000)]),
                    heads, kv_heads, hd, dtype, rng.random() < 0.5, pad)
    elif op == "attend":
        if rng.random() < 0.6:  # single tokens, and the few rows of a draft that is verified
            rows, length = rng.choice([1, 1, 1, 2, 3, 5, 8]), _log(rng, 1, 32700)
            seqs = _log(rng, 1, max(1, min(256, 8 * 256 * 4099 // (length * rows * kv_heads))))
        else:
            rows = _log(rng, 9, 1500)
            length = rows + rng.choice([0, _log(rng, 1, 2500)])
            seqs = _log(rng, 1, max(1, min(40, 12000000 // (rows * length))))
        c = _attend("", seqs, rows, length, rng.choice([0, 0, 0, _log(rng, 1, 2000)]), heads, kv_heads, hd, dtype, pad)
    else:
        vocab = _log(rng, 2, 200000)
        rows = _log(rng, 1, max(1, min(512, 128 * 151936 // vocab)))
        c = _sample("", rows, vocab, dtype, rng.choice([0, 1, 50, _log(rng, 1, vocab)]),
                    rng.choice([1.0, 0.95, 0.8, round(rng.uniform(0.05, 0.999), 4)]),
                    rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.0, 0.3), 4)]), rng.choice([1.0, 2.5, 4.0]))
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _below(g, n, *shape):
    return torch.randint(0, n, shape, generator=g, device="cuda")


def _pool(case, g, per_seq):
    """A pool whose pages belong to the sequences in mixed order, filled the
    way quantised keys and values fill it (the largest of a block near 127)."""
    kvh, hd, n_pages = case["kv_heads"], case["hd"], case["seqs"] * per_seq + 3
    codes = torch.empty(n_pages, 2, kvh, PAGE, hd, dtype=torch.int8, device="cuda")
    for a in range(0, n_pages, 8192):
        part = codes[a:a + 8192]
        part.copy_(_normal(g, *part.shape).mul_(36.0).round_().clamp_(-127, 127))
    scales = torch.exp(0.5 * _normal(g, n_pages, 2, kvh)) / 36.0
    order = torch.randperm(n_pages, generator=g, device="cuda")[:case["seqs"] * per_seq]
    return codes, scales, order.reshape(case["seqs"], per_seq).to(torch.int32)


def _rows(case, g, last):
    """seq and pos of a grid of seqs x rows that ends at each sequence's last
    position; a ragged sequence's missing rows, and `pad` rows behind all of
    them, are padding (seq -1)."""
    seqs, rows = case["seqs"], case["rows"]
    seq = torch.arange(seqs, device="cuda")[:, None].expand(seqs, rows).clone()
    pos = last[:, None] - (rows - 1) + torch.arange(rows, device="cuda")[None]
    if rows > 8:  # sequences of unlike length: the first one keeps all its rows
        have = rows - _below(g, rows // 2, seqs)
        have[0] = rows
        seq[torch.arange(rows, device="cuda")[None] >= have[:, None]] = -1
    pad = torch.full((case["pad"],), -1, device="cuda")
    return torch.cat([seq.reshape(-1), pad]).to(torch.int32), torch.cat([pos.reshape(-1), pad]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {"case": dict(case)}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (_normal(g, rows, vocab) * case["spread"]).to(TYPES[case["dtype"]])
        s["logits"][:, _below(g, vocab, max(1, vocab // 50))] = -math.inf  # tokens a grammar or a mask forbids
        s["temperature"] = 0.6 + 0.6 * torch.rand(rows, generator=g, device="cuda")
        s["temperature"][5::16] = 0.0  # greedy rows of a mixed batch
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        s["top_p"] = torch.full((rows,), case["top_p"], device="cuda")
        s["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["token"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["kept"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["logprob"] = torch.zeros(rows, device="cuda")
        return s
    heads, kvh, hd, dtype = case["heads"], case["kv_heads"], case["hd"], TYPES[case["dtype"]]
    if op == "append":
        start = case["start"] - _below(g, max(1, case["start"] // 2), case["seqs"])
        start[0] = case["start"]
        last = start + case["rows"] - 1
        top = case["start"] + case["rows"]
    else:
        last = case["length"] - 1 - (_below(g, max(1, case["length"] // 2), case["seqs"]) if case["rows"] <= 8 else
                                     _below(g, max(1, (case["length"] - case["rows"]) // 2), case["seqs"]))
        last[0] = case["length"] - 1
        top = case["length"]
    s["codes"], s["scales"], s["table"] = _pool(case, g, -(-top // PAGE))
    s["seq"], s["pos"] = _rows(case, g, last)
    n = s["seq"].numel()
    s["q"] = _normal(g, n, heads * hd).to(dtype)
    s["out"] = torch.zeros(n, heads * hd, dtype=dtype, device="cuda")
    if op == "append":
        s["k"], s["v"] = _normal(g, n, kvh * hd).to(dtype), _normal(g, n, kvh * hd).to(dtype)
        angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))[None]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = (1.0 + 0.1 * _normal(g, hd)).to(torch.float16)
            s["k_norm"] = (1.0 + 0.1 * _normal(g, hd)).to(torch.float16)
    else:
        s["lse"] = torch.zeros(n, heads, device="cuda")
    if own:  # the cache's description, which a program makes once with its buffers
        s["cache"] = _library().Kv8Cache(s["codes"].data_ptr(), s["scales"].data_ptr(), s["table"].data_ptr(),
                                         s["codes"].shape[0], case["seqs"], s["table"].shape[1], kvh, hd)
    return s


# ---- one pass ------------------------------------------------------------------


def run(s):
    return {"append": _run_append, "attend": _run_attend, "sample": _run_sample}[s["case"]["op"]](s)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _run_append(s):
    c = s["case"]
    if own:
        _library().kv8_append_dev(
            s["cache"], _ptr(s["k"]), _ptr(s["v"]), _ptr(s["seq"]), _ptr(s["pos"]), s["seq"].numel(),
            dtype=c["dtype"], q_ptr=_ptr(s["q"]), q_out_ptr=_ptr(s["out"]), heads=c["heads"],
            q_norm_ptr=_ptr(s["q_norm"]), k_norm_ptr=_ptr(s["k_norm"]), cos_ptr=_ptr(s["cos"]),
            sin_ptr=_ptr(s["sin"]), rope_rows=s["cos"].shape[0])
    else:
        _plain_append(s)
    return {"codes": s["codes"], "scales": s["scales"], "q": s["out"]}


def _run_attend(s):
    c = s["case"]
    if own:
        _library().kv8_attention_dev(
            s["cache"], _ptr(s["q"]), _ptr(s["out"]), _ptr(s["seq"]), _ptr(s["pos"]), s["seq"].numel(), c["heads"],
            dtype=c["dtype"], scale=1.0 / math.sqrt(c["hd"]), window=c["window"], max_rows=c["rows"],
            max_len=c["length"], lse_ptr=_ptr(s["lse"]))
    else:
        _plain_attend(s)
    return {"out": s["out"], "lse": s["lse"]}


def _run_sample(s):
    c = s["case"]
    if own:
        _library().sample_rows_dev(
            _ptr(s["logits"]), c["rows"], c["vocab"], _ptr(s["u"]), _ptr(s["token"]), dtype=c["dtype"],
            temperature_ptr=_ptr(s["temperature"]), top_k_ptr=_ptr(s["top_k"]), top_p_ptr=_ptr(s["top_p"]),
            min_p_ptr=_ptr(s["min_p"]), kept_ptr=_ptr(s["kept"]), logprob_ptr=_ptr(s["logprob"]))
        return {"token": s["token"], "kept": s["kept"], "logprob": s["logprob"]}
    return _plain_sample(s)


def _norm_rotate(x, gamma, cos, sin):
    """x [n][heads][hd] f32: RMS norm with its mean of squares summed in 64
    bits, then the rotation of the two halves, each step rounded in 32 bits."""
    if gamma is not None:
        mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
        x = x * (1.0 / torch.sqrt(mean + 1e-6)) * gamma.float()
    a, b = x.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    kvh, hd, codes, scales = c["kv_heads"], c["hd"], s["codes"], s["scales"]
    live = s["seq"] >= 0
    seq, pos = s["seq"][live].long(), s["pos"][live].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _norm_rotate(s["q"][live].float().reshape(-1, c["heads"], hd), s["q_norm"], cos, sin)
    s["out"][live] = q.reshape(q.shape[0], -1).to(s["out"].dtype)
    k = _norm_rotate(s["k"][live].float().reshape(-1, kvh, hd), s["k_norm"], cos, sin)
    kv = torch.stack([k, s["v"][live].float().reshape(-1, kvh, hd)], 1)  # [n][2][kv_heads][hd]
    page, slot = s["table"][seq, pos // PAGE].long(), pos % PAGE
    # the rows of one page form a block: its largest value and its first slot
    blocks, block = torch.unique(page, return_inverse=True)
    big = torch.zeros(len(blocks), 2, kvh, device="cuda")
    big.scatter_reduce_(0, block[:, None, None].expand(-1, 2, kvh), kv.abs().amax(-1), "amax")
    first = torch.full((len(blocks),), PAGE, device="cuda", dtype=torch.long)
    first.scatter_reduce_(0, block, slot, "amin")
    need = torch.where(big > 0, (big * (1.0 / 127.0)).clamp_min(2.0 ** -126), big)
    had = scales[blocks]
    new = torch.where((first == 0)[:, None, None], need, torch.where(need <= had, had, torch.maximum(need, had * 1.25)))
    ratio = torch.where(new > 0, had / new, torch.zeros_like(new))
    held = codes[blocks]
    again = (held.float() * ratio[..., None, None]).round().to(torch.int8)
    before = torch.arange(PAGE, device="cuda")[None] < first[:, None]
    codes[blocks] = torch.where(before[:, None, None, :, None], again, held)
    scales[blocks] = new
    inverse = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))[block]
    codes[page, :, :, slot] = (kv * inverse[..., None]).round().clamp(-127, 127).to(torch.int8)


def _visible(pos, length, window):
    at = torch.arange(length, device="cuda")
    seen = at <= pos[..., None]
    return seen & (at > pos[..., None] - window) if window else seen


def _plain_attend(s):
    c = s["case"]
    B, R, H, kvh, hd = c["seqs"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    length = s["table"].shape[1] * PAGE
    kv = s["codes"][s["table"].long()].float() * s["scales"][s["table"].long()][..., None, None]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, B, kvh, length, hd)  # [K|V][seq][kv_head][position][hd]
    q = s["q"][:B * R].float().reshape(B, R, kvh, H // kvh, hd).permute(0, 2, 3, 1, 4).reshape(B, kvh, -1, hd)
    score = torch.matmul(q, kv[0].transpose(-1, -2)).reshape(B, kvh, H // kvh, R, length) / math.sqrt(hd)
    seen = _visible(s["pos"][:B * R].reshape(B, R), length, c["window"])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(B, kvh, -1, length), kv[1]).reshape(B, kvh, H // kvh, R, hd)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    live = s["seq"][:B * R] >= 0
    s["out"][:B * R][live] = out.permute(0, 3, 1, 2, 4).reshape(B * R, H * hd).to(s["out"].dtype)[live]
    s["lse"][:B * R][live] = (torch.log(total) + top).permute(0, 3, 1, 2, 4).reshape(B * R, H)[live]


def _plain_sample(s):
    logits = s["logits"].float()
    logits = torch.where(torch.isnan(logits), torch.full_like(logits, -math.inf), logits)
    top = logits.amax(-1, keepdim=True)
    heat = s["temperature"].double()[:, None]
    greedy = ~(heat > 0)
    # weights and their sums in 64 bits: a draw is decided by a border of the running sum
    z = (logits.double() - top.double()) / torch.where(greedy, torch.ones_like(heat), heat)
    w = torch.where(logits == top, torch.ones_like(z), torch.exp(z))
    w = torch.where(logits == -math.inf, torch.zeros_like(w), w)
    _, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ws = w.gather(-1, order)
    rank = torch.arange(logits.shape[1], device="cuda")[None]
    k = s["top_k"][:, None]
    keep = (rank < k) | (k <= 0)
    ws = ws * keep
    p = s["top_p"].double()[:, None]
    keep &= (ws.cumsum(-1) - ws < p * ws.sum(-1, keepdim=True)) | (rank == 0) | ~(p < 1)
    keep &= (ws >= s["min_p"].double()[:, None].clamp(0, 1)) & (logits.gather(-1, order) > -math.inf)
    keep &= (rank == 0) | ~greedy
    kept = torch.zeros_like(keep).scatter_(-1, order, keep)
    run_sum = (w * kept).cumsum(-1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    token = torch.minimum(token, torch.where(kept, rank, torch.zeros_like(rank)).amax(-1, keepdim=True))
    logprob = torch.log(w.gather(-1, token) / total).float()
    count = kept.sum(-1).to(torch.int32)
    logprob = torch.where(count[:, None] > 0, logprob, torch.full_like(logprob, -math.inf))
    token = torch.where(count[:, None] > 0, token, torch.full_like(token, -1))
    return {"token": token[:, 0].to(torch.int32), "kept": count, "logprob": logprob[:, 0]}


# ---- what one pass cannot do without --------------------------------------------


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 4 * case["rows"] * case["vocab"]}
    hd, heads, kvh = case["hd"], case["heads"], case["kv_heads"]
    rows = case["seqs"] * case["rows"]
    ragged = 0.75 if case["rows"] > 8 else 1.0  # the mean share of a ragged sequence's rows
    if op == "append":
        rows = max(1.0, rows * ragged)
        moved = 2 * heads * hd * size + 2 * kvh * hd * size + 2 * kvh * hd
        held = case["seqs"] * 2 * kvh * (PAGE // 2) * hd  # the tokens before the first one in its page
        return {"bytes": rows * (moved + 2 * hd * 2) + held, "flops": rows * (heads + kvh) * hd * 6}
    first = case["length"] - case["rows"]
    if case["rows"] <= 8:
        lengths = 0.75 * case["length"]
    else:
        lengths = 0.75 * first + case["rows"]
    window = case["window"] or 1 << 30
    seen = min(lengths, window + case["rows"] - 1)
    pairs = rows * ragged * min(max(1.0, lengths - case["rows"] / 2.0), window)
    return {"bytes": case["seqs"] * seen * kvh * 2 * hd + rows * ragged * heads * hd * 2 * size,
            "flops": 4.0 * pairs * heads * hd}


# ---- the same from the definitions, in 64 bits -----------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_heads(x, heads, gamma, s, pos):
    x = x.double().reshape(x.shape[0], heads, -1)
    if gamma is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * gamma.double()
    half = x.shape[-1] // 2
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_append(s):
    """Queries and scales; a code is a rounding to 8 bits of a value rounded
    in 32, so it has no value of its own in 64."""
    c = s["case"]
    rows = torch.nonzero(s["seq"] >= 0)[:, 0]
    pos = s["pos"][rows].long()
    out = s["out"].double()
    out[rows] = _exact_heads(s["q"][rows], c["heads"], s["q_norm"], s, pos).reshape(len(rows), -1)
    k = _exact_heads(s["k"][rows], c["kv_heads"], s["k_norm"], s, pos).abs().amax(-1)
    v = s["v"][rows].double().reshape(k.shape[0], c["kv_heads"], -1).abs().amax(-1)
    need = (torch.stack([k, v], 1) / 127.0).cpu().numpy()
    page = s["table"][s["seq"][rows].long(), pos // PAGE].cpu().numpy()
    slot = (pos % PAGE).cpu().numpy()
    scales = s["scales"].double().cpu().numpy()
    old, seen = scales.copy(), {}
    for i, at in enumerate(page):  # rows of a page come in the order of their slots
        if at not in seen:
            seen[at] = (slot[i] == 0, need[i])
        else:
            seen[at] = (seen[at][0], np.maximum(seen[at][1], need[i]))
    for at, (fresh, most) in seen.items():
        scales[at] = most if fresh else np.where(most <= old[at], old[at], np.maximum(most, 1.25 * old[at]))
    return {"codes": None, "scales": torch.from_numpy(scales), "q": out}


def _exact_attend(s):
    c = s["case"]
    H, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
    out, lse = s["out"].double(), s["lse"].double()
    seq_host = s["seq"].cpu()
    for b in range(c["seqs"]):
        rows = torch.nonzero(seq_host == b)[:, 0].cuda()
        if not len(rows):
            continue
        pages = s["table"][b].long()
        kv = s["codes"][pages].double() * s["scales"][pages].double()[..., None, None]
        at = torch.arange(len(pages) * PAGE, device="cuda")[None]
        pos = s["pos"][rows].long()[:, None]
        hidden = (at > pos) | ((at <= pos - c["window"]) if c["window"] else (at < 0))
        for h in range(H):
            k, v = (kv[:, i, h * kvh // H].reshape(-1, hd) for i in (0, 1))
            a = s["q"][rows, h * hd:(h + 1) * hd].double() @ k.T / math.sqrt(hd)
            a[hidden] = -math.inf
            norm = torch.logsumexp(a, -1)
            seen = norm > -math.inf
            got = torch.exp(a - torch.where(seen, norm, torch.zeros_like(norm))[:, None]) @ v
            out[rows, h * hd:(h + 1) * hd] = got
            lse[rows, h] = norm
    return {"out": out, "lse": lse}


def _exact_sample(s):
    rows, vocab = s["logits"].shape
    token, kept, logprob = np.full(rows, -1), np.zeros(rows, np.int64), np.full(rows, -math.inf)
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    heat, u = s["temperature"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    top_k, top_p, min_p = (s[n].cpu().numpy() for n in ("top_k", "top_p", "min_p"))
    for r in range(rows):
        x = logits[r]
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -math.inf]
        if not len(order):
            continue
        if not heat[r] > 0:
            token[r], kept[r], logprob[r] = order[0], 1, 0.0
            continue
        if top_k[r] > 0:
            order = order[:top_k[r]]
        w = np.exp((x[order] - x[order[0]]) / heat[r])
        total = math.fsum(w)
        n = len(order)
        if top_p[r] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w)[:-1], float(top_p[r]) * total))
        n = min(n, int((w >= float(min_p[r])).sum()))
        back = np.argsort(order[:n])
        total = math.fsum(w[:n])
        i = min(int(np.searchsorted(np.cumsum(w[:n][back]), u[r] * total, side="right")), n - 1)
        token[r], kept[r] = order[:n][back][i], n
        logprob[r] = math.log(w[:n][back][i] / total)
    return {"token": torch.from_numpy(token).to(torch.int32), "kept": torch.from_numpy(kept).to(torch.int32),
            "logprob": torch.from_numpy(logprob)}
