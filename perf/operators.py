"""The operators of a hybrid model's softmax-attention layers, as a user's program
calls them next to the delta-rule layers: rotary positions, the paged key/value
cache that is appended to, attention over it, and causal attention in training.

A case is a dict of plain values:

  op           "rotary" (queries and keys rotated; "train": with the gradient),
               "append" (keys, rotated, and values into a paged cache),
               "paged" (attention of new tokens over a paged cache),
               "train" (causal attention forward and backward)
  dtype        "bf16", "f16" or "f32"
  B            sequences (rows)
  T            most new tokens of a sequence; training and rotary: tokens per row
  ctx          append, paged: most cached tokens of a sequence before the new ones
  ragged       append, paged: sequences differ in new and in cached tokens
  Hq, Hkv, D   query heads, key/value heads, channels of a head
  R            rotary, append: channels that are rotated
  interleaved  rotary, append: pairs (2i, 2i + 1) instead of (i, i + R/2)
  page         tokens of a cache page
  heads_first  append, paged: a page is stored (head, token, channel)
  window       tokens that a query sees, itself among them; 0 for all before it
  doc          rotary, training: mean document length of packed rows, 0 for one document

``own`` False: the plain form in elementary torch operations; True: the calls of
this package.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _api():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "deltanet-tpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import deltanet_tpu_amd
    return deltanet_tpu_amd


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rotary(B, T, Hq, Hkv, D, R, dtype="bf16", interleaved=False, train=False, doc=0):
    return dict(op="rotary", dtype=dtype, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, R=R, interleaved=interleaved, train=train, doc=doc)


def _append(B, T, ctx, Hkv, D, R, page, dtype="bf16", interleaved=False, ragged=False, heads_first=False):
    return dict(op="append", dtype=dtype, B=B, T=T, ctx=ctx, ragged=ragged, Hkv=Hkv, D=D, R=R, interleaved=interleaved,
                page=page, heads_first=heads_first)


def _paged(B, T, ctx, Hq, Hkv, D, page, dtype="bf16", ragged=False, heads_first=False, window=0):
    return dict(op="paged", dtype=dtype, B=B, T=T, ctx=ctx, ragged=ragged, Hq=Hq, Hkv=Hkv, D=D, page=page,
                heads_first=heads_first, window=window)


def _train(B, T, Hq, Hkv, D, dtype="bf16", doc=0, window=0):
    return dict(op="train", dtype=dtype, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, doc=doc, window=window)


def listed():
    return [
        # one token of 64 sequences, a quarter of each head rotated
        dict(_rotary(64, 1, 16, 4, 256, 64), name="rotary-64"),
        # a training batch's queries and keys and their gradients, packed documents
        dict(_rotary(2, 4096, 32, 8, 128, 128, train=True, doc=1024), name="rotary-train-2x4096"),
        # one token of 64 sequences stored
        dict(_append(64, 1, 500, 4, 256, 64, 64), name="append-64"),
        # prompts of up to 2048 tokens stored behind what is cached, small pages
        dict(_append(16, 2048, 1024, 8, 128, 128, 16, interleaved=True, ragged=True, heads_first=True), name="append-16x2048"),
        # one user's token after a short prompt
        dict(_paged(1, 1, 1000, 16, 4, 256, 64), name="decode-1x1000"),
        # a full serving batch, contexts of very different length
        dict(_paged(64, 1, 16384, 32, 8, 128, 64, ragged=True), name="decode-64x16384"),
        # drafts of 5 tokens verified for 32 sequences
        dict(_paged(32, 5, 4096, 16, 4, 256, 16, dtype="f16", ragged=True), name="draft-32x5"),
        # prompts in chunks next to sequences that are nearly done, a sliding window
        dict(_paged(12, 777, 3000, 16, 4, 128, 64, ragged=True, window=1024), name="mixed-12x777"),
        # the second half of two prompts over the first one, cached
        dict(_paged(2, 4096, 4096, 16, 4, 256, 128), name="prompt-2x4096"),
        # training in float32 at a ragged length, as many key heads as query heads
        dict(_train(2, 300, 8, 8, 64, dtype="f32"), name="train-2x300-f32"),
        # training at the ordinary prompt's size, two documents or so
        dict(_train(1, 2048, 16, 4, 256, doc=1024), name="train-2048"),
        # a large batch of long rows
        dict(_train(2, 8192, 16, 4, 128), name="train-2x8192"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "paged", "paged", "paged", "train", "train"])
    Hq, Hkv = rng.choice([(16, 4), (16, 2), (32, 8), (8, 8), (24, 4), (5, 1)])
    D = rng.choice([64, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    R = rng.choice([D, D, D // 2, D // 4])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if op == "rotary":
        B = _log_int(rng, 1, 64)
        return _rotary(B, _log_int(rng, 1, max(2, 8000 // B)), Hq, Hkv, D, R, dtype, rng.random() < 0.5, rng.random() < 0.5,
                       rng.choice([0, 128, 1024]))
    if op == "append":
        B = _log_int(rng, 1, 64)
        return _append(B, _log_int(rng, 1, max(2, 16000 // B)), _log_int(rng, 1, 1000), Hkv, D, R, page, dtype,
                       rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.3)
    window = rng.choice([0, 0, 0, 100, 1024])
    if op == "paged":
        kind = rng.choice(["decode", "draft", "chunk"])
        B = _log_int(rng, 1, 64 if kind != "chunk" else 8)
        T = {"decode": 1, "draft": rng.randint(2, 16), "chunk": _log_int(rng, 17, max(18, 4000 // B))}[kind]
        # a quarter of the largest listed cases' cached values at most
        most = (1 << 28) // (B * Hkv * D) if kind != "chunk" else 8192 // B
        return _paged(B, T, _log_int(rng, 16, max(17, min(most, 20000))), Hq, Hkv, D, page, dtype, rng.random() < 0.7,
                      rng.random() < 0.3, window)
    B = rng.choice([1, 1, 2, 3, 4])
    most = (4096 if dtype == "f32" or D == 256 else 6000) // B
    return _train(B, _log_int(rng, 16, most), Hq, Hkv, D, dtype, rng.choice([0, 0, 128, 1024]), window)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case):
    """(new tokens, cached tokens) of each sequence: all alike, or spread evenly
    over the range, short and long ones mixed."""
    B = case["B"]
    if not case["ragged"]:
        return [case["T"]] * B, [case["ctx"]] * B
    u = [((i + 1) * 0.6180339887) % 1.0 for i in range(B)]
    w = [((i + 1) * 0.7548776662) % 1.0 for i in range(B)]
    new = [max(1, int(round(case["T"] * x * x))) for x in w]
    new[0] = case["T"]
    old = [int(round(case["ctx"] * x)) for x in u]
    old[B // 2] = case["ctx"]
    return new, old


def _starts(case, seed):
    """First token (B, T) of each token's document, lengths geometric, at least 16."""
    rng = np.random.default_rng(seed)
    B, T = case["B"], case["T"]
    start = np.zeros((B, T), np.int64)
    if case["doc"]:
        for b in range(B):
            t = 0
            while t < T:
                n = int(max(rng.geometric(1.0 / case["doc"]), 16))
                start[b, t:t + n] = t
                t += n
    return torch.from_numpy(start).cuda()


def _table(positions, R):
    """cos and sin of position * 10000^(-2i/R): (positions, R), computed in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([torch.cos(a), torch.sin(a)], dim=1).to(torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    dt, B, T, D, Hkv = DTYPES[case["dtype"]], case["B"], case["T"], case["D"], case["Hkv"]
    s = {"case": case}
    if case["op"] == "rotary":
        Hq = case["Hq"]
        # queries, keys and values of one projection, side by side
        qkv = rn(B, T, Hq + 2 * Hkv, D).to(dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        t = torch.arange(T, device="cuda")
        if T == 1:  # decoding: every sequence at a place of its own
            s["pos"] = torch.randint(0, 8192, (B, 1), device="cuda", generator=gen)
            s["table"] = _table(8192, case["R"])
        else:
            s["pos"] = t[None, :] - _starts(case, seed)
            s["table"] = _table(T, case["R"])
        if case["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
            s["dq"], s["dk"] = rn(B, T, Hq, D).to(dt), rn(B, T, Hkv, D).to(dt)
        return s
    if case["op"] == "train":
        Hq = case["Hq"]
        s["q"], s["k"], s["v"] = rn(B, T, Hq, D).to(dt), rn(B, T, Hkv, D).to(dt), rn(B, T, Hkv, D).to(dt)
        s["do"] = rn(B, T, Hq, D).to(dt)
        s["leaves"] = [s[n].requires_grad_(True) for n in ("q", "k", "v")]
        s["start"] = _starts(case, seed)
        s["seg"] = s["start"].to(torch.int32) if case["doc"] else None
        return s
    rng = np.random.default_rng(seed)
    new, old = _lens(case)
    order = rng.permutation(B)
    new, old = np.asarray(new)[order], np.asarray(old)[order]
    lens, page = new + old, case["page"]
    counts = -(-lens // page)
    most, pages = int(counts.max()), int(counts.sum()) + 2
    free = rng.permutation(pages)
    table = np.zeros((B, most), np.int32)
    at = 0
    for b in range(B):
        table[b, :counts[b]] = free[at:at + counts[b]]
        at += counts[b]
    cu = np.concatenate([[0], np.cumsum(new)])
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", torch.int32)
    s["pages"], s["lens"], s["cu"] = dev(table), dev(lens), dev(cu)
    n = int(cu[-1])
    for name in ("kc", "vc"):
        if case["heads_first"]:
            s[name] = rn(pages, Hkv, page, D).to(dt).transpose(1, 2)
        else:
            s[name] = rn(pages, page, Hkv, D).to(dt)
    if case["op"] == "append":
        s["k"], s["v"] = rn(n, Hkv, D).to(dt), rn(n, Hkv, D).to(dt)
        s["table"] = _table(case["ctx"] + T, case["R"])
    else:
        s["q"] = rn(n, case["Hq"], D).to(dt)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rotated(x, rows, R, interleaved, back=False):
    """x (..., H, D) in 32 bits with its first R channels rotated by rows (..., R) of the table."""
    c, s = rows[..., None, :R // 2], rows[..., None, R // 2:]
    if back:
        s = -s
    x = x.to(torch.float32)
    r = x[..., :R]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    y = (a * c - b * s, b * c + a * s)
    y = torch.stack(y, dim=-1).flatten(-2) if interleaved else torch.cat(y, dim=-1)
    return torch.cat([y, x[..., R:]], dim=-1)


def _scores(q, k, first, last, scale):
    """Probabilities (B, Hkv, G T, S) of q (B, Hkv, G T, D) over k (B, Hkv, S, D); a query sees keys first .. last
    (B, T each) and a query without any has zeros."""
    G = q.shape[2] // first.shape[1]
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j >= first[..., None]) & (j <= last[..., None])
    seen = seen.repeat(1, G, 1)[:, None]
    x = torch.matmul(q, k.transpose(2, 3)) * scale
    x = torch.where(seen, x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    return x / x.sum(-1, keepdim=True).clamp_min(1e-30)


def _grouped(x, Hkv):
    """(B, T, Hq, D) as (B, Hkv, G T, D) in 32 bits."""
    B, T, H, D = x.shape
    return x.to(torch.float32).reshape(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)


def _ungrouped(x, T):
    B, H, n, D = x.shape
    return x.reshape(B, H, n // T, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H * (n // T), D)


def _first(start, last, window):
    return torch.maximum(start, last - window + 1) if window else start


def _places(s, n):
    """Sequence, place among its new tokens and position of each of n new tokens."""
    cu, lens = s["cu"].long(), s["lens"].long()
    i = torch.arange(n, device=cu.device)
    b = torch.searchsorted(cu, i, right=True) - 1
    return b, i - cu[b], lens[b] - (cu[b + 1] - i)


def _plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        dt, rows = s["q"].dtype, s["table"][s["pos"]]
        turn = lambda x, back: _rotated(x, rows, c["R"], c["interleaved"], back).to(dt)
        out = [turn(s["q"].detach(), False), turn(s["k"].detach(), False)]
        return out + [turn(s["dq"], True), turn(s["dk"], True)] if c["train"] else out
    if c["op"] == "append":
        b, _, pos = _places(s, s["k"].shape[0])
        at = (s["pages"].long()[b, pos // c["page"]], pos % c["page"])
        s["kc"][at] = _rotated(s["k"], s["table"][pos], c["R"], c["interleaved"]).to(s["kc"].dtype)
        s["vc"][at] = s["v"]
        return [s["kc"], s["vc"]]
    scale = 1.0 / math.sqrt(c["D"])
    if c["op"] == "paged":
        q, Hkv, T = s["q"], c["Hkv"], c["T"]
        b, i, pos = _places(s, q.shape[0])
        all_q = torch.zeros((c["B"], T) + q.shape[1:], dtype=torch.float32, device=q.device)
        all_q[b, i] = q.to(torch.float32)
        last = torch.full((c["B"], T), -1, dtype=torch.int64, device=q.device)
        last[b, i] = pos
        rows = lambda x: x[s["pages"].long()].flatten(1, 2).to(torch.float32).transpose(1, 2)
        p = _scores(_grouped(all_q, Hkv), rows(s["kc"]), _first(torch.zeros_like(last), last, c["window"]), last, scale)
        return _ungrouped(torch.matmul(p, rows(s["vc"])), T)[b, i].to(q.dtype)
    q, k, v = (_grouped(s[n].detach(), c["Hkv"]) for n in ("q", "k", "v"))
    do, dt, T = _grouped(s["do"], c["Hkv"]), s["q"].dtype, c["T"]
    last = torch.arange(T, device=q.device).expand(c["B"], T)
    p = _scores(q, k, _first(s["start"], last, c["window"]), last, scale)
    o = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    return [_ungrouped(o, T).to(dt), [_ungrouped(x, T).to(dt) for x in (dq, dk, dv)]]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    if not own:
        with torch.no_grad():
            return _plain(s)
    m, c = _api(), s["case"]
    if c["op"] == "rotary":
        q, k = m.apply_rotary(s["q"], s["k"], s["pos"], s["table"], interleaved=c["interleaved"])
        if not c["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    if c["op"] == "append":
        m.paged_kv_append(s["k"], s["v"], s["kc"], s["vc"], s["pages"], s["lens"], cu_seqlens=s["cu"], table=s["table"],
                          interleaved=c["interleaved"])
        return [s["kc"], s["vc"]]
    if c["op"] == "paged":
        return m.paged_attention(s["q"], s["kc"], s["vc"], s["pages"], s["lens"], cu_seqlens=s["cu"],
                                 window=c["window"] or None)
    out = m.causal_attention(s["q"], s["k"], s["v"], segment_ids=s["seg"], window=c["window"] or None)
    return [out.detach(), list(torch.autograd.grad(out, s["leaves"], s["do"]))]


def _pairs(case):
    """Pairs of a query and a key that it sees, per query head; training without documents."""
    w = case["window"] or 1 << 60
    full = lambda n: n * (n + 1) // 2
    below = lambda n: full(n) - full(max(0, n - w))  # tokens 0 .. n-1 of one sequence, window applied
    if case["op"] == "train":
        n, d = case["T"], case["doc"]
        if not d or d >= n:
            return case["B"] * below(n)
        return case["B"] * (n // d * below(d) + below(n % d))
    new, old = _lens(case)
    return sum(below(n + o) - below(o) for n, o in zip(new, old))


def work(case):
    """Inputs read once and outputs written once; for attention the products of
    every pair that is seen: two forward, and five more backward (the
    probabilities come again from the scores there)."""
    e, D, Hkv = (4 if case["dtype"] == "f32" else 2), case["D"], case["Hkv"]
    if case["op"] == "rotary":
        x = case["B"] * case["T"] * (case["Hq"] + Hkv)
        both = 2 if case["train"] else 1
        table = case["B"] * case["T"] * (4 * case["R"] + 8)
        return {"bytes": float(both * (2 * x * D * e + table)), "flops": 3.0 * both * x * case["R"]}
    if case["op"] == "append":
        n = sum(_lens(case)[0])
        return {"bytes": float(n * (4 * Hkv * D * e + 4 * case["R"])), "flops": 3.0 * n * Hkv * case["R"]}
    Hq, pairs = case["Hq"], _pairs(case)
    if case["op"] == "paged":
        new, old = _lens(case)
        w = case["window"] or 1 << 60
        cached = sum(min(n + o, n + w - 1) for n, o in zip(new, old))
        return {"bytes": float(e * D * (2 * cached * Hkv + 2 * sum(new) * Hq)), "flops": 4.0 * pairs * Hq * D}
    n = case["B"] * case["T"]
    # forward: q, k, v, out; backward: those and out's gradient again, three gradients
    return {"bytes": float(e * n * D * (2 * Hq + 2 * Hkv + 4 * Hq + 4 * Hkv)), "flops": 14.0 * pairs * Hq * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _turn64(x, pos, table, R, interleaved):
    """x (N, H, D) times the rotation matrices, as complex numbers."""
    z = torch.complex(table[pos, :R // 2].double(), table[pos, R // 2:].double())[:, None]
    y = x.double().clone()
    if interleaved:
        y[..., :R] = torch.view_as_real(torch.view_as_complex(y[..., :R].reshape(*y.shape[:-1], R // 2, 2).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(y[..., :R // 2].contiguous(), y[..., R // 2:R].contiguous()) * z
        y[..., :R // 2], y[..., R // 2:R] = w.real, w.imag
    return y


def _attend64(q, k, v, hidden, scale):
    x = (q @ k.T) * scale
    return torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    D, scale = case["D"], 1.0 / math.sqrt(case["D"])
    if case["op"] == "rotary":
        flat = lambda x: x.detach().flatten(0, 1)
        pos, inv = s["pos"].flatten(), s["table"].clone()
        inv[:, case["R"] // 2:] *= -1.0
        turn = lambda n, t: _turn64(flat(s[n]), pos, t, case["R"], case["interleaved"]).reshape(s[n].shape)
        out = [turn("q", s["table"]), turn("k", s["table"])]
        return out + [turn("dq", inv), turn("dk", inv)] if case["train"] else out
    if case["op"] in ("append", "paged"):
        cu, lens, pages = s["cu"].tolist(), s["lens"].tolist(), s["pages"].long()
    if case["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        for b in range(case["B"]):
            pos = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda")
            at = (pages[b, pos // case["page"]], pos % case["page"])
            new = slice(cu[b], cu[b + 1])
            kc[at] = _turn64(s["k"][new], pos, s["table"], case["R"], case["interleaved"])
            vc[at] = s["v"][new].double()
        return [kc, vc]
    G, w = case["Hq"] // case["Hkv"], case["window"] or 1 << 60
    if case["op"] == "paged":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            j = torch.arange(lens[b], device="cuda")
            i = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda")[:, None]
            hidden = (j > i) | (j <= i - w)
            at = (pages[b, j // case["page"]], j % case["page"])
            k, v, q = s["kc"][at].double(), s["vc"][at].double(), s["q"][cu[b]:cu[b + 1]].double()
            for h in range(case["Hq"]):
                out[cu[b]:cu[b + 1], h] = _attend64(q[:, h], k[:, h // G], v[:, h // G], hidden, scale)
        return out
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "do"))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(case["T"], device="cuda")
    for b in range(case["B"]):
        hidden = (j > j[:, None]) | (j <= j[:, None] - w) | (j < s["start"][b][:, None])
        for h in range(case["Hq"]):
            part = [x.contiguous().requires_grad_(True) for x in (q[b, :, h], k[b, :, h // G], v[b, :, h // G])]
            y = _attend64(*part, hidden, scale)
            g = torch.autograd.grad(y, part, do[b, :, h].contiguous())
            o[b, :, h], dq[b, :, h] = y.detach(), g[0]
            dk[b, :, h // G] += g[1]
            dv[b, :, h // G] += g[2]
    return [o, [dq, dk, dv]]
