"""The operators around a hybrid model's softmax-attention layers that a server
with drafted trees and a trainer with normed heads call: norms of queries and keys
with their rotation, the same with the store into a paged cache, page tables and
slots from the requests' lengths, attention of drafted trees, and the accepted
path's tokens moved to the front.

A case is a dict of plain values:

  op           "norm" (queries and keys normed and rotated, with all gradients),
               "append" (the same for serving: queries out, keys and values into a paged cache),
               "step" (pages reserved, slots mapped, pages given back),
               "tree" (attention of drafted trees over a paged cache),
               "keep" (the accepted path moved to the front, all layers)
  dtype        "bf16", "f16" or "f32"
  wide         norm: the norms' weights are float32 whatever the dtype
  B            sequences (rows)
  T            most new tokens of a sequence; norm: tokens per row
  ctx          most cached tokens of a sequence before the new ones
  ragged       sequences differ in new and in cached tokens
  trees        step: the new tokens are drafted trees
  Hq, Hkv, D   query heads, key/value heads, channels of a head
  R            channels that are rotated
  interleaved  pairs (2i, 2i + 1) instead of (i, i + R/2)
  page         tokens of a cache page
  heads_first  a page is stored (head, token, channel)
  window       tree: tokens that a query sees; 0 for all
  layers       keep: layers of the cache

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
EPS, OFFSET = 1e-6, 1.0   # the norms' weights are kept as differences from 1


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

def _norm(B, T, Hq, Hkv, D, R, dtype="bf16", wide=False, interleaved=False):
    return dict(op="norm", dtype=dtype, wide=wide, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, R=R, interleaved=interleaved)


def _append(B, T, ctx, Hq, Hkv, D, R, page, dtype="bf16", interleaved=False, ragged=False, heads_first=False):
    return dict(op="append", dtype=dtype, B=B, T=T, ctx=ctx, ragged=ragged, Hq=Hq, Hkv=Hkv, D=D, R=R,
                interleaved=interleaved, page=page, heads_first=heads_first)


def _step(B, T, ctx, page, ragged=False, trees=False):
    return dict(op="step", B=B, T=T, ctx=ctx, page=page, ragged=ragged, trees=trees)


def _tree(B, T, ctx, Hq, Hkv, D, page, dtype="bf16", ragged=False, heads_first=False, window=0):
    return dict(op="tree", dtype=dtype, B=B, T=T, ctx=ctx, ragged=ragged, Hq=Hq, Hkv=Hkv, D=D, page=page,
                heads_first=heads_first, window=window)


def _keep(B, T, ctx, layers, Hkv, D, page, dtype="bf16", ragged=False, heads_first=False):
    return dict(op="keep", dtype=dtype, B=B, T=T, ctx=ctx, layers=layers, Hkv=Hkv, D=D, page=page, ragged=ragged,
                heads_first=heads_first)


def listed():
    return [
        # a training batch's queries and keys, with the gradients of the norms' weights
        dict(_norm(2, 4096, 32, 8, 128, 128), name="norm-2x4096"),
        # a small float32 batch of ragged length, a quarter of each head rotated
        dict(_norm(3, 301, 16, 4, 256, 64, dtype="f32", interleaved=True), name="norm-3x301-f32"),
        # one token of 64 sequences
        dict(_append(64, 1, 500, 16, 4, 256, 64, 64), name="append-64"),
        # prompts of up to 2048 tokens behind what is cached, small pages
        dict(_append(16, 2048, 1024, 32, 8, 128, 128, 16, interleaved=True, ragged=True, heads_first=True), name="append-16x2048"),
        # the bookkeeping of one token of 64 sequences
        dict(_step(64, 1, 500, 64, ragged=True), name="step-64"),
        # of a full batch of drafted trees, trimmed to what was accepted
        dict(_step(64, 33, 4096, 16, ragged=True, trees=True), name="step-trees-64x33"),
        # of a long queue of prompts, admitted and released
        dict(_step(2048, 8192, 0, 16, ragged=True), name="step-2048x8192"),
        # one user's small tree after a short prompt
        dict(_tree(1, 16, 1000, 16, 4, 256, 64), name="tree-1x16"),
        # trees of a serving batch, small pages
        dict(_tree(32, 25, 4096, 16, 4, 256, 16, dtype="f16", ragged=True), name="tree-32x25-f16"),
        # large trees over long contexts
        dict(_tree(16, 64, 16384, 32, 8, 128, 64, ragged=True), name="tree-16x64"),
        # one user's accepted tokens, in every layer
        dict(_keep(1, 16, 1000, 12, 4, 256, 64), name="keep-1x16"),
        # a serving batch's
        dict(_keep(64, 33, 500, 12, 8, 128, 16, ragged=True), name="keep-64x33"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "append", "step", "step", "tree", "tree", "tree", "keep"])
    Hq, Hkv = rng.choice([(16, 4), (16, 2), (32, 8), (8, 8), (24, 4), (5, 1)])
    D = rng.choice([64, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    R = rng.choice([D, D, D // 2, D // 4])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    B = _log_int(rng, 1, 64)
    if op == "norm":
        return _norm(B, _log_int(rng, 1, max(2, 8000 // B)), Hq, Hkv, D, R, dtype, rng.random() < 0.3, rng.random() < 0.5)
    if op == "append":
        return _append(B, _log_int(rng, 1, max(2, 16000 // B)), _log_int(rng, 1, 1000), Hq, Hkv, D, R, page, dtype,
                       rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.3)
    if op == "step":
        trees = rng.random() < 0.5
        B = _log_int(rng, 1, 256 if trees else 2048)
        T = _log_int(rng, 2, 200 if trees else 8192)
        return _step(B, T, _log_int(rng, 1, 8000), page, rng.random() < 0.8, trees)
    if op == "tree":
        B, T = _log_int(rng, 1, 48), _log_int(rng, 2, 128)
        most = min((1 << 28) // (B * Hkv * D), (1 << 33) // (B * T * Hq * D), 20000)
        return _tree(B, T, _log_int(rng, 16, max(17, most)), Hq, Hkv, D, page, dtype, rng.random() < 0.7,
                     rng.random() < 0.3, rng.choice([0, 0, 0, 1024]))
    return _keep(B, _log_int(rng, 4, 64), _log_int(rng, 1, 500), rng.choice([1, 4, 12]), Hkv, D, page, dtype, rng.random() < 0.8,
                 rng.random() < 0.3)


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


def _shuffled_lens(case, rng):
    order = rng.permutation(case["B"])
    new, old = _lens(case)
    return np.asarray(new, np.int64)[order], np.asarray(old, np.int64)[order]


def _parents(new, rng):
    """Each new token's parent among its sequence's, -1 for children of the cached
    text: trees laid down level by level, narrow ones and wide ones."""
    out = []
    for n in new:
        wide = rng.integers(1, 6)
        lo, hi, level = -1, 0, []   # the level above: [lo, hi)
        while len(level) < n:
            size = min(n - len(level), int(wide))
            above = [-1] * size if lo < 0 else sorted(rng.integers(lo, hi, size))
            lo, hi = len(level), len(level) + size
            level += [int(x) for x in above]
        out += level
    return np.asarray(out, np.int32)


def _pages(lens, page, rng, spare=2):
    """A page table of permuted pages for sequences of these lengths, and the number of pages."""
    counts = -(-lens // page)
    pages = int(counts.sum()) + spare
    table = np.zeros((len(lens), max(int(counts.max()), 1)), np.int32)
    free = rng.permutation(pages)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = free[at:at + c]
        at += c
    return table, pages


def _table(positions, R):
    """cos and sin of position * 10000^(-2i/R): (positions, R), computed in 64 bits."""
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([torch.cos(a), torch.sin(a)], dim=1).to(torch.float32)


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _ancestors(parents, new):
    """(sum of n, most) truth values on the host: which of its sequence's new tokens each sees."""
    most, at, rows = int(max(new)), 0, []
    for n in new:
        m = np.zeros((n, most), bool)
        for i, p in enumerate(parents[at:at + n]):
            if p >= 0:
                m[i] = m[p]
            m[i, i] = True
        rows.append(m)
        at += n
    return np.concatenate(rows)


def _words(m):
    """Truth values (N, n) as (N, ceil(n / 64)) 64-bit words, the lowest bit first."""
    m = np.pad(m, ((0, 0), (0, -m.shape[1] % 64)))
    return np.packbits(m, axis=1, bitorder="little").view(np.int64)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    s, B, T = {"case": case}, case["B"], case["T"]
    if case["op"] == "norm":
        dt, D, Hq, Hkv = DTYPES[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
        # queries, keys and values of one projection, side by side
        qkv = rn(B, T, Hq + 2 * Hkv, D).to(dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        wt = torch.float32 if case["wide"] else dt
        s["wq"], s["wk"] = (0.2 * rn(D)).to(wt), (0.2 * rn(D)).to(wt)
        s["leaves"] = [s[n].detach().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
        s["dq"], s["dk"] = rn(B, T, Hq, D).to(dt), rn(B, T, Hkv, D).to(dt)
        s["pos"], s["table"] = torch.arange(T, device="cuda"), _table(T, case["R"])
        return s
    new, old = _shuffled_lens(case, rng)
    cu = np.concatenate([[0], np.cumsum(new)])
    n, page = int(cu[-1]), case["page"]
    s["n"], s["cu"] = n, _dev(cu)
    if case["op"] == "step":
        held = -(-old // page)
        table, pages = _pages(old, page, rng, spare=int((-(-(old + new) // page) - held).sum()) + 3)
        used = np.concatenate([table[b, :h] for b, h in enumerate(held)])
        free = rng.permutation(np.setdiff1d(np.arange(pages), used))
        most = int((-(-(old + new) // page)).max())
        s["pages"] = _dev(np.pad(table, ((0, 0), (0, max(0, most - table.shape[1])))))
        # the pool: the number of free pages, a word of the kernel's, the pages
        s["pool"] = _dev(np.concatenate([[len(free), 0], free, np.zeros(pages - len(free), np.int64)]))
        s["held"], s["old"], s["lens"] = _dev(held), _dev(old), _dev(old + new)
        s["parents"] = _dev(_parents(new, rng)) if case["trees"] else None
        return s
    dt, D, Hkv = DTYPES[case["dtype"]], case["D"], case["Hkv"]
    table, pages = _pages(old + new, page, rng)
    s["pages"], s["lens"] = _dev(table), _dev(old + new)
    lead = (case["layers"],) if case["op"] == "keep" else ()
    for name in ("kc", "vc"):
        if case["heads_first"]:
            s[name] = torch.stack([rn(pages, Hkv, page, D).to(dt) for _ in range(lead[0] if lead else 1)])
            s[name] = s[name].transpose(2, 3)
        else:
            s[name] = torch.stack([rn(pages, page, Hkv, D).to(dt) for _ in range(lead[0] if lead else 1)])
        if not lead:
            s[name] = s[name][0]
    if case["op"] == "append":
        q = rn(n, case["Hq"] + 2 * Hkv, D).to(dt)
        s["q"], s["k"], s["v"] = q[:, :case["Hq"]], q[:, case["Hq"]:-Hkv], q[:, -Hkv:]
        s["wq"], s["wk"] = (0.2 * rn(D)).to(dt), (0.2 * rn(D)).to(dt)
        s["table"] = _table(case["ctx"] + T, case["R"])
        b = np.repeat(np.arange(B), new)
        at = old[b] + np.arange(n) - cu[b]
        s["pos"], s["slots"] = _dev(at), _dev(table[b, at // page].astype(np.int64) * page + at % page, torch.int64)
    elif case["op"] == "tree":
        s["q"] = rn(n, case["Hq"], D).to(dt)
        s["visible"] = _dev(_words(_ancestors(_parents(new, rng), new)), torch.int64)
    else:
        # the first drafted token and some of those far behind it: what a pass moves
        # it does not overwrite, so that it can be repeated
        kept = np.full((B, 8), -1)
        for b in range(B):
            m = int(min(rng.integers(1, 9), (new[b] + 1) // 2))
            kept[b, :m] = np.concatenate([[0], np.sort(rng.choice(np.arange(m, new[b]), m - 1, replace=False))]) if m > 1 else 0
        s["kept"], s["start"] = _dev(kept), _dev(old)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rotated(x, rows, R, interleaved, back=False):
    """x (..., H, D) in 32 bits with its first R channels rotated by rows (..., R) of the table."""
    c, s = rows[..., None, :R // 2], rows[..., None, R // 2:]
    if back:
        s = -s
    r = x[..., :R]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    y = (a * c - b * s, b * c + a * s)
    y = torch.stack(y, dim=-1).flatten(-2) if interleaved else torch.cat(y, dim=-1)
    return torch.cat([y, x[..., R:]], dim=-1)


def _normed(x, w):
    """x over its root mean square, with the weights and without, and what it was multiplied by."""
    x = x.to(torch.float32)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r * (OFFSET + w.to(torch.float32)), x * r, r


def _plain_norm(s):
    c, rows, out, grads, dw = s["case"], s["table"][s["pos"]], [], [], []
    for x, w, dz in ((s["q"], s["wq"], s["dq"]), (s["k"], s["wk"], s["dk"])):
        y, u, r = _normed(x, w)
        out.append(_rotated(y, rows, c["R"], c["interleaved"]).to(x.dtype))
        g = _rotated(dz.to(torch.float32), rows, c["R"], c["interleaved"], back=True)
        h = g * (OFFSET + w.to(torch.float32))
        grads.append((r * (h - u * (h * u).mean(-1, keepdim=True))).to(x.dtype))
        dw.append((g * u).double().sum((0, 1, 2)).to(w.dtype))
    return out + grads + dw


def _plain_append(s):
    c, rows = s["case"], s["table"][s["pos"].long()]
    turn = lambda x, w: _rotated(_normed(x, w)[0], rows, c["R"], c["interleaved"])
    at = (s["slots"] // c["page"], s["slots"] % c["page"])
    s["kc"][at] = turn(s["k"], s["wk"]).to(s["kc"].dtype)
    s["vc"][at] = s["v"]
    return [turn(s["q"], s["wq"]).to(s["q"].dtype), s["kc"], s["vc"]]


def _plain_reserve(pool, table, held, lens, page):
    """Pages given back, then taken, as a stack; the pages that each sequence is short of."""
    col = torch.arange(table.shape[1], device=table.device)
    need, h = (lens.long().clamp_min(0) + page - 1) // page, held.long()
    freed, grow = (h - need).clamp_min(0), (need - h).clamp_min(0)
    count, most = pool[0].long(), pool.shape[0] - 2
    # the last page of the last sequence first
    behind = freed.sum() - torch.cumsum(freed, 0)
    back = (col >= need[:, None]) & (col < h[:, None])
    to = count + behind[:, None] + (h[:, None] - 1 - col)
    stack = torch.cat([pool[2:], pool[:1]])   # (and a place for what is not pushed)
    stack.scatter_(0, torch.where(back, to, most).flatten(), table.flatten())
    full = count + freed.sum()
    upto = torch.cumsum(grow, 0)
    fits = upto <= full
    grow = torch.where(fits, grow, 0)
    before = torch.cumsum(grow, 0) - grow
    new = torch.where(freed > 0, need, h + grow)
    take = (col >= h[:, None]) & (col < new[:, None])
    at = (full - 1 - before[:, None] - (col - h[:, None])).clamp(0, most - 1)
    table.copy_(torch.where(take, stack[at], table))
    pool[2:] = stack[:-1]
    pool[0] = full - grow.sum()
    held.copy_(new)
    return (need - new).clamp_min(0).to(torch.int32)


def _places(cu, lens, n):
    """Sequence, place among its new tokens and slot's position of each of n new tokens."""
    cu, lens = cu.long(), lens.long()
    i = torch.arange(n, device=cu.device)
    b = torch.searchsorted(cu, i, right=True) - 1
    return b, i - cu[b], lens[b] - (cu[b + 1] - i)


def _plain_slots(s):
    c, page = s["case"], s["case"]["page"]
    b, i, at = _places(s["cu"], s["lens"], s["n"])
    slots = s["pages"].long()[b, at // page] * page + at % page
    if s["parents"] is None:
        return [at.to(torch.int32), slots]
    # ancestors: products of truth values, the number of generations doubled each time
    T = c["T"]
    sees = torch.eye(T, device="cuda").repeat(c["B"], 1, 1)
    parent = s["parents"].long()
    sees[b, i, parent.clamp_min(0)] = torch.where(parent < 0, sees[b, i, parent.clamp_min(0)], 1.0)
    for _ in range(max(1, (T - 1).bit_length())):
        sees = (torch.matmul(sees, sees) > 0).to(torch.float32)
    seen = sees[b, i] > 0
    depth = seen.sum(-1) - 1
    seen = torch.cat([seen, seen.new_zeros(seen.shape[0], -T % 64)], dim=1).reshape(seen.shape[0], -1, 64)
    words = (seen.long() << torch.arange(64, device="cuda")).sum(-1)
    return [(at - i + depth).to(torch.int32), slots, words]


def _plain_step(s):
    page = s["case"]["page"]
    short = _plain_reserve(s["pool"], s["pages"], s["held"], s["lens"], page)
    out = _plain_slots(s)
    less = _plain_reserve(s["pool"], s["pages"], s["held"], s["old"], page)
    return [s["pages"], short, *out, less, s["held"], s["pool"]]


def _grouped(x, Hkv):
    """(B, T, Hq, D) as (B, Hkv, G T, D) in 32 bits."""
    B, T, H, D = x.shape
    return x.to(torch.float32).reshape(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)


def _ungrouped(x, T):
    B, H, n, D = x.shape
    return x.reshape(B, H, n // T, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H * (n // T), D)


def _plain_tree(s):
    c, q, Hkv, B, T = s["case"], s["q"], s["case"]["Hkv"], s["case"]["B"], s["case"]["T"]
    b, i, _ = _places(s["cu"], s["lens"], s["n"])
    all_q = torch.zeros((B, T) + q.shape[1:], dtype=torch.float32, device=q.device)
    all_q[b, i] = q.to(torch.float32)
    words = torch.zeros((B, T, s["visible"].shape[1]), dtype=torch.int64, device=q.device)
    words[b, i] = s["visible"]
    bits = ((words[..., None] >> torch.arange(64, device=q.device)) & 1).flatten(2) > 0
    rows = lambda x: x[s["pages"].long()].flatten(1, 2).to(torch.float32).transpose(1, 2)
    k, v = rows(s["kc"]), rows(s["vc"])
    j = torch.arange(k.shape[2], device=q.device)
    cached = (s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None, None]
    rel = (j - cached).expand(B, T, -1)
    seen = torch.where(rel < 0, True, torch.gather(bits, 2, rel.clamp(0, bits.shape[2] - 1)) & (rel < bits.shape[2]))
    if c["window"]:
        seen = seen & ((rel >= 0) | (j >= cached + bits.sum(-1, keepdim=True) - c["window"]))
    seen = seen.repeat(1, c["Hq"] // Hkv, 1)[:, None]
    x = torch.matmul(_grouped(all_q, Hkv), k.transpose(2, 3)) * (1.0 / math.sqrt(c["D"]))
    x = torch.where(seen, x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
    return _ungrouped(torch.matmul(x, v), T)[b, i].to(q.dtype)


def _plain_keep(s):
    page, kept, start = s["case"]["page"], s["kept"].long(), s["start"].long()
    on = kept >= 0
    lens = start + on.sum(1)
    here = lambda at: (torch.gather(s["pages"].long(), 1, at // page), at % page)
    to = start[:, None] + torch.arange(kept.shape[1], device="cuda")
    # tokens that are not kept are written onto the first one that is
    from_ = start[:, None] + torch.where(on, kept, kept[:, :1])
    to = torch.where(on, to, start[:, None])
    (tp, to), (fp, from_) = here(to), here(from_)
    for x in (s["kc"], s["vc"]):
        x[:, tp, to] = x[:, fp, from_]
    return [s["kc"], s["vc"], lens.to(torch.int32)]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_PLAIN = {"norm": _plain_norm, "append": _plain_append, "step": _plain_step, "tree": _plain_tree, "keep": _plain_keep}


def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return _PLAIN[c["op"]](s)
    m = _api()
    if c["op"] == "norm":
        q, k = m.norm_rotary(*s["leaves"], s["pos"], s["table"], eps=EPS, weight_offset=OFFSET, interleaved=c["interleaved"])
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"]))]
    if c["op"] == "append":
        q = m.paged_qkv_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["pos"], q_weight=s["wq"],
                               k_weight=s["wk"], eps=EPS, weight_offset=OFFSET, table=s["table"], interleaved=c["interleaved"])
        return [q, s["kc"], s["vc"]]
    if c["op"] == "step":
        page = c["page"]
        short = m.paged_reserve(s["pool"], s["pages"], s["held"], s["lens"], page_size=page)
        out = m.paged_slots(s["pages"], s["lens"], s["n"], page_size=page, cu_seqlens=s["cu"], parents=s["parents"],
                            nodes=c["T"] if c["trees"] else None)
        less = m.paged_reserve(s["pool"], s["pages"], s["held"], s["old"], page_size=page)
        return [s["pages"], short, *out, less, s["held"], s["pool"]]
    if c["op"] == "tree":
        return m.paged_tree_attention(s["q"], s["kc"], s["vc"], s["pages"], s["lens"], s["visible"], cu_seqlens=s["cu"],
                                      window=c["window"] or None)
    lens = m.paged_kv_keep(s["kc"], s["vc"], s["pages"], s["start"], s["kept"])
    return [s["kc"], s["vc"], lens]


def work(case):
    """Inputs read once and outputs written once; what a pass does not touch of a
    cache, a page table or a pool is not counted."""
    new, old = _lens(case) if case["op"] != "norm" else ([case["T"]] * case["B"], None)
    n = sum(new)
    if case["op"] == "step":
        page = case["page"]
        taken = sum(-(-(a + b) // page) - -(-b // page) for a, b in zip(new, old))
        # pages out of the pool into the table, both ways; lengths and counts; positions, slots, pages read; trees
        words = 8 * -(-case["T"] // 64) + 4 if case["trees"] else 0
        return {"bytes": float(16 * taken + 28 * case["B"] + n * (12 + words) + 4 * (n // page)), "flops": float(n)}
    e, D, Hkv = (4 if case["dtype"] == "f32" else 2), case["D"], case["Hkv"]
    if case["op"] == "norm":
        x, table = n * (case["Hq"] + Hkv), n * 4 * case["R"]
        # forward: in, out; backward: in and gradient, gradient out
        return {"bytes": float(x * D * e * 5 + 2 * table), "flops": float(x * (16 * D + 6 * case["R"]))}
    if case["op"] == "append":
        x = n * (case["Hq"] + 2 * Hkv)
        return {"bytes": float(2 * x * D * e + n * (4 * case["R"] + 12)), "flops": float(n * (case["Hq"] + Hkv) * (4 * D + 3 * case["R"]))}
    if case["op"] == "tree":
        w = case["window"] or 1 << 60
        seen = [min(o, w) for o in old]   # of the cached tokens, about
        pairs = sum(a * (o + min(a, 8)) for a, o in zip(new, seen))
        return {"bytes": float(e * D * (2 * Hkv * (sum(seen) + n) + 2 * n * case["Hq"])), "flops": 4.0 * pairs * case["Hq"] * D}
    # between 1 and 8 kept tokens of a sequence, all but the first moved
    moved = sum(min(3.5, (a + 1) // 2 - 1) for a in new)
    return {"bytes": float(4 * moved * Hkv * D * e * case["layers"] + 44 * case["B"]), "flops": 0.0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _turn64(x, pos, table, R, interleaved):
    """x (N, H, D) times the rotation matrices, as complex numbers."""
    z = torch.complex(table[pos, :R // 2].double(), table[pos, R // 2:].double())[:, None]
    if interleaved:
        y = torch.view_as_real(torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * z
        y = torch.cat([w.real, w.imag], dim=-1)
    return torch.cat([y, x[..., R:]], dim=-1)


def _norm64(x, w):
    x = x.double()
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (OFFSET + w.double())


def _exact_step(case, s):
    """The stack and the trees walked through on the host."""
    page = case["page"]
    pool, held, cu = s["pool"].tolist(), s["held"].tolist(), s["cu"].tolist()
    table = s["pages"].cpu().numpy().copy()
    count, stack = pool[0], pool[2:]

    def reserve(lens):
        nonlocal count
        need, short, enough = [-(-x // page) for x in lens], [], True
        for b in reversed(range(case["B"])):
            while held[b] > need[b]:
                held[b] -= 1
                stack[count] = int(table[b, held[b]])
                count += 1
        for b in range(case["B"]):
            enough = enough and need[b] - held[b] <= count
            while enough and held[b] < need[b]:
                count -= 1
                table[b, held[b]] = stack[count]
                held[b] += 1
            short.append(need[b] - held[b])
        return short

    new, old = s["lens"].tolist(), s["old"].tolist()
    first = reserve(new)
    out = [np.zeros(s["n"], np.int64), np.zeros(s["n"], np.int64)]
    seen = None
    if s["parents"] is not None:
        parents = s["parents"].cpu().numpy()
        seen = _ancestors(parents, np.diff(cu))
        if seen.shape[1] < case["T"]:
            seen = np.pad(seen, ((0, 0), (0, case["T"] - seen.shape[1])))
    for b in range(case["B"]):
        at = np.arange(old[b], new[b])
        rows = slice(cu[b], cu[b + 1])
        out[0][rows] = at if seen is None else old[b] + seen[rows].sum(1) - 1
        out[1][rows] = table[b, at // page].astype(np.int64) * page + at % page
    if seen is not None:
        out.append(_words(seen))
    second = reserve(old)
    out = [table, first, *out, second, held, [count, 0] + stack]
    return [torch.from_numpy(np.asarray(x, np.int64)).cuda() for x in out]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        return _exact_step(case, s)
    if case["op"] == "norm":
        leaves = [x.detach().double().contiguous().requires_grad_(True) for x in s["leaves"]]
        pos = s["pos"].repeat(case["B"])
        turn = lambda x, w: _turn64(_norm64(x, w).flatten(0, 1), pos, s["table"], case["R"], case["interleaved"]).reshape(x.shape)
        q, k = turn(leaves[0], leaves[2]), turn(leaves[1], leaves[3])
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["dq"].double(), s["dk"].double()))]
    if case["op"] == "append":
        turn = lambda x, w: _turn64(_norm64(x, w), s["pos"].long(), s["table"], case["R"], case["interleaved"])
        kc, vc, k = s["kc"].double(), s["vc"].double(), turn(s["k"], s["wk"])
        at = (s["slots"] // case["page"], s["slots"] % case["page"])
        kc[at], vc[at] = k, s["v"].double()
        return [turn(s["q"], s["wq"]), kc, vc]
    if case["op"] == "keep":
        kc, vc = s["kc"].double(), s["vc"].double()
        pages, lens = s["pages"].tolist(), s["start"].tolist()
        put = lambda b, p: (pages[b][p // case["page"]], p % case["page"])
        for b, row in enumerate(s["kept"].tolist()):
            for i, x in enumerate(row):
                if x < 0:
                    break
                (tp, t), (fp, f) = put(b, lens[b]), put(b, lens[b] - i + x)
                for c in (kc, vc):
                    c[:, tp, t] = c[:, fp, f].clone()
                lens[b] += 1
        return [kc, vc, torch.tensor(lens, device="cuda")]
    cu, lens, pages = s["cu"].tolist(), s["lens"].tolist(), s["pages"].long()
    G, w, page = case["Hq"] // case["Hkv"], case["window"] or 1 << 60, case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    words = s["visible"].cpu().numpy().view(np.uint8)
    bits = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")).cuda() > 0
    for b in range(case["B"]):
        n = cu[b + 1] - cu[b]
        j = torch.arange(lens[b], device="cuda")
        mine = bits[cu[b]:cu[b + 1], :n]
        hidden = torch.cat([torch.zeros(n, lens[b] - n, dtype=torch.bool, device="cuda"), ~mine], dim=1)
        # of the tokens that a row sees, those with `window` or more behind them
        hidden |= (~hidden).flip(1).cumsum(1).flip(1) > w
        at = (pages[b, j // page], j % page)
        k, v, q = s["kc"][at].double(), s["vc"][at].double(), s["q"][cu[b]:cu[b + 1]].double()
        for h in range(case["Hq"]):
            x = (q[:, h] @ k[:, h // G].T) / math.sqrt(case["D"])
            out[cu[b]:cu[b + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // G]
    return out
