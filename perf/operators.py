"""The operators of a paged KV cache and of beam search, as cases that can be timed and checked.

A case is a dict of plain values; `prepare` makes on the GPU what a program holds before the call, `run`
makes one pass and returns its whole outputs, `exact` gives them in float64.  With `own` false `run`
computes in elementary torch operations, with `own` true through this framework's entry points.

Kinds (field "kind"):
  attention  new tokens of a ragged batch (a chunk of a prompt, or one token each) over a paged cache
  write      the new tokens' K and V rows into their pages
  step       the pages of a beam search step: rows follow their parents, grow by a token, and shared
             tail pages are copied for their new owners
  compact    live pages moved to the front of the pool
  select     the best continuations of every beam group over beams x vocabulary

The cache: page pools [pages, kv heads, page size, head dim], a page table [sequences, table width] of
page ids (-1: none) and the number of cached rows of each sequence, the new tokens' among them.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # Serving eight long conversations: one token each over 8k to 32k cached rows (the largest reads).
        {"name": "decode_bf16_8x32768", "kind": "attention", "dtype": "bfloat16", "batch": 8, "hq": 16, "hkv": 8, "d": 128,
         "page": 16, "new": 1, "len": 32768, "shared": 0, "evicted": False},
        # Two short chats from float32 pages: the smallest attention call.
        {"name": "decode_f32_2x777", "kind": "attention", "dtype": "float32", "batch": 2, "hq": 16, "hkv": 8, "d": 128,
         "page": 16, "new": 1, "len": 777, "shared": 0, "evicted": False},
        # A beam search step: four prompts of eight beams each that share their prompt's pages.
        {"name": "decode_bf16_beams_32x1531", "kind": "attention", "dtype": "bfloat16", "batch": 32, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "new": 1, "len": 1531, "shared": 8, "evicted": False},
        # Chunked prefill of a long prompt: 2048 new tokens behind 14336 cached rows.
        {"name": "chunk_bf16_1x2048_of_16384", "kind": "attention", "dtype": "bfloat16", "batch": 1, "hq": 16, "hkv": 8,
         "d": 128, "page": 64, "new": 2048, "len": 16384, "shared": 0, "evicted": False},
        # A mixed serving batch: ragged chunks, short and long, at odd lengths.
        {"name": "chunk_bf16_6x300_of_2600", "kind": "attention", "dtype": "bfloat16", "batch": 6, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "new": 300, "len": 2600, "shared": 0, "evicted": False},
        # The same on the float32-activation path, which is the model's default.
        {"name": "chunk_f32_2x200_of_1000", "kind": "attention", "dtype": "float32", "batch": 2, "hq": 16, "hkv": 8,
         "d": 128, "page": 32, "new": 200, "len": 1000, "shared": 0, "evicted": False},
        # A long chunk's rows into their pages (memory bound), and one token of eight sequences (latency).
        {"name": "write_bf16_4x2048", "kind": "write", "dtype": "bfloat16", "batch": 4, "hkv": 8, "d": 128, "page": 16,
         "new": 2048, "len": 4096},
        {"name": "write_f32_8x1", "kind": "write", "dtype": "float32", "batch": 8, "hkv": 8, "d": 128, "page": 16, "new": 1,
         "len": 1000},
        # One beam step of eight prompts with eight beams over a cache of eight layers.
        {"name": "step_bf16_8x8", "kind": "step", "dtype": "bfloat16", "groups": 8, "beams": 8, "layers": 8, "hkv": 8, "d": 128,
         "page": 16, "len": 1000},
        # A fragmented pool of four layers after many sequences ended.
        {"name": "compact_bf16_4000", "kind": "compact", "dtype": "bfloat16", "sequences": 48, "layers": 4, "hkv": 8, "d": 128,
         "page": 16, "pages": 4000},
        # One prompt with four beams over the model's vocabulary; and sixteen with eight, from bfloat16 logits.
        {"name": "select_f32_1x4", "kind": "select", "dtype": "float32", "groups": 1, "beams": 4, "vocab": 151936,
         "finished": False},
        {"name": "select_bf16_16x8", "kind": "select", "dtype": "bfloat16", "groups": 16, "beams": 8, "vocab": 151936,
         "finished": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "write", "step", "compact", "select", "select"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "attention":
        hq, hkv = rng.choice([(16, 8), (32, 8), (40, 8), (16, 16)])
        case = {"kind": kind, "dtype": dtype, "hq": hq, "hkv": hkv, "d": rng.choice([128, 128, 64]), "page": page,
                "shared": 0, "evicted": rng.random() < 0.2}
        if rng.random() < 0.5:
            shared = rng.choice([0, 0, 4, 8])
            batch = shared * rng.randint(1, 4) if shared else _log(rng, 1, 48)
            most = min(32768, (130000 if dtype == "bfloat16" else 65000) * 8 // (batch * hkv))
            return {**case, "batch": batch, "new": 1, "len": _log(rng, 100, max(200, most)), "shared": shared}
        new = _log(rng, 2, 2048 if dtype == "bfloat16" else 512)
        batch = rng.randint(1, 8)
        # no more pairs of tokens and keys than the largest listed chunk (float32: a fraction of them)
        pairs = 2048 * 16384 * 16 // (batch * hq) // (1 if dtype == "bfloat16" else 8)
        new = min(new, math.isqrt(pairs))
        return {**case, "batch": batch, "new": new, "len": new + _log(rng, 1, max(2, min(16000 // batch, pairs // new - new)))}
    if kind == "write":
        batch = rng.randint(1, 8)
        new = _log(rng, 1, 8192 // batch)
        return {"kind": kind, "dtype": dtype, "batch": batch, "hkv": 8, "d": rng.choice([128, 64]), "page": page, "new": new,
                "len": new + rng.randint(0, 2000)}
    if kind == "step":
        return {"kind": kind, "dtype": dtype, "groups": rng.randint(1, 8), "beams": rng.randint(2, 8),
                "layers": rng.randint(1, 4), "hkv": 8, "d": rng.choice([128, 64]), "page": rng.choice([16, 32]),
                "len": _log(rng, 20, 1500)}
    if kind == "compact":
        return {"kind": kind, "dtype": dtype, "sequences": rng.randint(1, 64), "layers": rng.randint(1, 2), "hkv": 8,
                "d": rng.choice([128, 64]), "page": rng.choice([16, 32]), "pages": _log(rng, 100, 2000)}
    return {"kind": kind, "dtype": dtype, "groups": rng.randint(1, 16), "beams": rng.randint(1, 8),
            "vocab": _log(rng, 1000, 151936), "finished": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------
# Inputs (from the seed alone)
# ---------------------------------------------------------------------------------------------
EOS = 7  # the end token's id of the select cases


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 27  # random numbers of at most half a GiB at a time
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda") * std
    return out


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _pages_of(lens, page):
    return -(-np.asarray(lens) // page)


def _geometry(case, seed):
    """New tokens and cached rows of each sequence, the page table, and the pool's size.  The lengths go by the
    case alone, their order and the pages by the seed."""
    b, new, most, page = case["batch"], case["new"], case["len"], case["page"]
    r = np.random.RandomState(most + 7 * b)
    n = np.full(b, new)
    if new > 1:  # some chunks shorter, one of them full
        n = r.randint(1, new + 1, size=b)
        n[r.randint(b)] = new
    lens = np.maximum(n, r.randint(max(1, most // 4), most + 1, size=b))
    at = r.randint(b)
    lens[at], n[at] = most, new
    group = case.get("shared", 0) or 1
    shared = np.zeros(b, np.int64)  # leading pages shared by the group
    if group > 1:
        for i in range(0, b, group):
            own_rows = 64
            base = max(1, int(lens[i:i + group].max()) - own_rows)
            lens[i:i + group] = base + r.randint(1, own_rows + 1, size=len(lens[i:i + group]))
            shared[i:i + group] = base // page
        lens = np.minimum(lens, most)
    r = np.random.RandomState(seed % (1 << 31))
    by = (r.permutation(b // group)[:, None] * group + r.permutation(group)[None]).reshape(-1)
    n, lens, shared = n[by], lens[by], shared[by]
    count = _pages_of(lens, page)
    width = int(count.max()) + 2
    rows = []
    total = 0
    for i in range(b):
        head = rows[i - i % group][:shared[i - i % group]] if i % group else []
        fresh = count[i] - len(head)
        rows.append(list(head) + list(range(total, total + fresh)))
        total += fresh
    pool = total + 3
    order = r.permutation(pool)
    table = np.full((b, width), -1, np.int64)
    for i in range(b):
        table[i, :count[i]] = order[np.asarray(rows[i], np.int64)]
        if case.get("evicted") and count[i] > 8:  # the middle is gone: the first page and the last ones stay
            table[i, 1:count[i] // 2] = -1
    return n.astype(np.int64), lens.astype(np.int64), table, pool


def _beam_pages(case, seed):
    """Page table, lengths, reference counts and parents of groups of beams that share their prompt."""
    page, beams, fixed = case["page"], case["beams"], np.random.RandomState(case["len"] + 7 * case["groups"])
    prompts = fixed.randint(max(1, case["len"] // 2), case["len"] + 1, size=case["groups"])
    tails = fixed.randint(1, 4 * page, size=case["groups"])  # rows that the beams wrote since
    r = np.random.RandomState(seed % (1 << 31))
    rows, lens, parents, total = [], [], [], 0
    for g in r.permutation(case["groups"]):
        prompt, tail = int(prompts[g]), int(tails[g])
        head = list(range(total, total + prompt // page))
        total += len(head)
        for _ in range(beams):
            count = -(-(prompt + tail) // page) - len(head)
            rows.append(head + list(range(total, total + count)))
            total += count
            lens.append(prompt + tail)
        parents += list(len(parents) + r.randint(0, beams, size=beams))
    s = len(rows)
    width = -(-max(lens) // page) + 2
    pool = total + 2 * s
    order = r.permutation(pool)
    table = np.full((s, width), -1, np.int64)
    refs = np.zeros(pool, np.int64)
    for i, row in enumerate(rows):
        ids = order[np.asarray(row, np.int64)]
        table[i, :len(ids)] = ids
        refs[ids] += 1
    return table, np.asarray(lens), refs, np.asarray(parents), pool


def _fragments(case, seed):
    """Page table and reference counts of sequences spread over a pool that is two fifths full."""
    pool, s = case["pages"], case["sequences"]
    live = np.random.RandomState(seed % (1 << 31)).permutation(pool)[: max(1, 2 * pool // 5)]
    cuts = np.sort(np.random.RandomState(pool + s).randint(0, len(live) + 1, size=s - 1))
    parts = np.split(live, cuts)
    width = max(len(p) for p in parts) + 1
    table = np.full((s, width), -1, np.int64)
    refs = np.zeros(pool, np.int64)
    for i, p in enumerate(parts):
        table[i, :len(p)] = p
        refs[p] += 1
    if s > 1:  # the second sequence shares the first one's leading pages
        n = min(len(parts[0]), len(parts[1]), 4)
        refs[table[1, :n]] -= 1
        table[1, :n] = table[0, :n]
        refs[table[0, :n]] += 1
    return table, refs


def _inputs(case, seed):
    """The case's tensors (a dict of torch tensors on the GPU)."""
    g, dt, kind = _gen(seed), _dt(case), case["kind"]
    if kind in ("attention", "write"):
        n, lens, table, pool = _geometry(case, seed)
        starts = np.concatenate([[0], np.cumsum(n)])
        shape = (pool, case["hkv"], case["page"], case["d"])
        x = {"kp": _randn(g, *shape, dtype=dt), "vp": _randn(g, *shape, dtype=dt), "table": _int(table), "lens": _int(lens)}
        if case["new"] > 1:
            x["starts"] = _int(starts)
        if kind == "attention":
            x["q"] = _randn(g, int(starts[-1]), case["hq"], case["d"], dtype=dt)
        else:
            x["k"] = _randn(g, int(starts[-1]), case["hkv"], case["d"], dtype=dt)
            x["v"] = _randn(g, int(starts[-1]), case["hkv"], case["d"], dtype=dt)
        return x
    if kind == "step":
        table, lens, refs, parents, pool = _beam_pages(case, seed)
        return {"table": _int(table), "lens": _int(lens), "refs": _int(refs), "parents": _int(parents),
                "counts": _int(np.ones(len(lens))),
                "pages": _randn(g, case["layers"], 2, pool, case["hkv"], case["page"], case["d"], dtype=dt)}
    if kind == "compact":
        table, refs = _fragments(case, seed)
        return {"table": _int(table), "refs": _int(refs),
                "pages": _randn(g, case["layers"], 2, case["pages"], case["hkv"], case["page"], case["d"], dtype=dt)}
    groups, beams = case["groups"], case["beams"]
    x = {"logits": _randn(g, groups, beams, case["vocab"], std=3.0, dtype=dt),
         "scores": -20 * torch.rand(groups, beams, generator=g, device="cuda")}
    if case["finished"]:
        x["finished"] = (torch.rand(groups, beams, generator=g, device="cuda") < 0.25).to(torch.int32)
    return x


# ---------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------
def _places(x, tokens):
    """Sequence and position of every token: the last n rows of a sequence are its new tokens."""
    lens = x["lens"].long()
    starts = x["starts"].long() if "starts" in x else torch.arange(len(lens) + 1, device="cuda")
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    j = t - starts[seq]
    n = starts[1:] - starts[:-1]
    return seq, j, lens[seq] - n[seq] + j, starts, n


def _plain_attention(x, case):
    q, table, lens, page = x["q"], x["table"].long(), x["lens"].long(), case["page"]
    b, tokens, hkv, d = case["batch"], q.shape[0], case["hkv"], case["d"]
    ratio, width, new = case["hq"] // hkv, -(-case["len"] // page), case["new"]
    table = table[:, :width]
    seq, j, pos, starts, n = _places(x, tokens)
    gathered = lambda p: p[table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(b, hkv, width * page, d).float()  # noqa: E731
    at = (starts[:-1, None] + torch.arange(new, device="cuda")).clamp(max=tokens - 1)
    rows = q[at].float().view(b, new, hkv, ratio, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, ratio * new, d)
    scores = torch.matmul(rows, gathered(x["kp"]).transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hkv, ratio, new, -1)
    key = torch.arange(width * page, device="cuda")
    there = (table >= 0).repeat_interleave(page, 1)
    last = (lens - n)[:, None] + torch.arange(new, device="cuda")  # the last key that each new token sees
    seen = (key <= last[..., None]) & there[:, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(p.view(b, hkv, ratio * new, -1), gathered(x["vp"]))
    o = o.view(b, hkv, ratio, new, d).permute(0, 3, 1, 2, 4).reshape(b, new, case["hq"], d)
    return o[seq, j].to(q.dtype)


def _plain_write(x, case):
    seq, _, pos, _, _ = _places(x, x["k"].shape[0])
    page, slot = x["table"].long()[seq, pos // case["page"]], pos % case["page"]
    x["kp"][page, :, slot] = x["k"]
    x["vp"][page, :, slot] = x["v"]
    return {"kp": x["kp"], "vp": x["vp"]}


def _count(table, pool, weight):
    """Sum of `weight` over the entries of a page table, by page."""
    held = table >= 0
    return torch.zeros(pool, dtype=torch.long, device="cuda").index_add_(
        0, table.clamp(min=0).reshape(-1), (held * weight).reshape(-1))


def _plain_step(x, case):
    page, s = case["page"], x["table"].shape[0]
    old, parents, refs, grow = x["table"].long(), x["parents"].long(), x["refs"].long(), x["counts"].long()
    pool, rows = refs.shape[0], torch.arange(s, device="cuda")
    # rows follow their parents
    table, lens = old[parents], x["lens"].long()[parents]
    children = torch.zeros(s, dtype=torch.long, device="cuda").index_add_(0, parents, torch.ones_like(parents))
    refs = refs + _count(old, pool, (children - 1)[:, None])
    # and grow: a shared tail page is copied, by every sharer or by all but the last
    tail = table.gather(1, (lens // page)[:, None])[:, 0]
    part = (lens % page != 0) & (grow > 0)
    same = (tail[:, None] == tail[None]) & part[:, None] & part[None]
    keeps = (refs[tail.clamp(min=0)] <= same.sum(1)) & ~(same & (rows[None] > rows[:, None])).any(1)
    copies = part & ~keeps
    first = (lens + page - 1) // page - copies.long()  # the first table entry that gets a new page
    need = (lens + grow + page - 1) // page - first
    before = need.cumsum(0) - need
    free = (refs == 0).nonzero()[:, 0]
    missing = (need.sum() - len(free)).clamp(min=0)
    at = torch.arange(table.shape[1], device="cuda")[None] - first[:, None]
    taken = (at >= 0) & (at < need[:, None])
    fresh = free[(before[:, None] + at).clamp(0, len(free) - 1)]
    moves = torch.full((s, 2), -1, dtype=torch.long, device="cuda")
    src, dst = tail[copies], fresh.gather(1, first[:, None])[:, 0][copies]
    moves[: len(src)] = torch.stack([src, dst], 1)
    table = torch.where(taken, fresh, table)
    refs = refs - torch.zeros_like(refs).index_add_(0, src, torch.ones_like(src))
    refs[table[taken]] = 1
    # the copied pages of every layer
    pages = x["pages"]
    pages[:, :, dst] = pages[:, :, src]
    info = torch.stack([copies.sum(), missing, torch.zeros_like(missing)])
    return {"table": table.int(), "lens": (lens + grow).int(), "refs": refs.int(), "moves": moves.int(), "info": info.int(),
            "pages": pages}


def _plain_compact(x, case):
    table, refs, pages = x["table"].long(), x["refs"].long(), x["pages"]
    pool = refs.shape[0]
    live = refs > 0
    count = live.sum()
    behind = torch.arange(pool, device="cuda") >= count
    src, dst = (live & behind).nonzero()[:, 0], (~live & ~behind).nonzero()[:, 0]
    to = torch.arange(pool, device="cuda")
    to[src] = dst
    moves = torch.full((max(1, pool // 2), 2), -1, dtype=torch.long, device="cuda")
    moves[: len(src)] = torch.stack([src, dst], 1)
    new = refs.clone()
    new[dst] = refs[src]
    new[src] = 0
    pages[:, :, dst] = pages[:, :, src]
    table = torch.where(table >= 0, to[table.clamp(min=0)], table)
    return {"table": table.int(), "refs": new.int(), "moves": moves.int(),
            "info": torch.stack([torch.full_like(count, len(src)), count]).int(), "pages": pages}


def _plain_select(x, case):
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    logits = x["logits"].double()  # sums of many terms, and values next to a border
    top = logits.amax(-1, keepdim=True)
    logits -= top + (logits - top).exp().sum(-1, keepdim=True).log()
    scores = logits + x["scores"].double()[..., None]
    if case["finished"]:  # a finished beam goes on as itself, with the end token
        done = x["finished"].bool()[..., None]
        only = torch.arange(vocab, device="cuda") == EOS
        scores = torch.where(done, torch.where(only, x["scores"].double()[..., None], -math.inf), scores)
    best, at = scores.view(groups, -1).sort(stable=True, dim=-1, descending=True)
    best, at = best[:, :beams], at[:, :beams]
    parents, tokens = at // vocab, at % vocab
    out = {"scores": best.float(), "tokens": tokens.int(), "parents": parents.int()}
    if case["finished"]:
        out["finished"] = (x["finished"].bool().gather(1, parents) | (tokens == EOS)).int()
    return out


# ---------------------------------------------------------------------------------------------
# The framework's tensors: filled from torch, and seen by it
# ---------------------------------------------------------------------------------------------
_NAME = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.int32: "int32"}
_CODE = {"float32": "<f4", "bfloat16": "<i2", "int32": "<i4"}


class _Device:
    """A contiguous tensor's device memory for torch.as_tensor (shared, not copied)."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": tuple(tensor.shape), "typestr": _CODE[tensor.dtype], "strides": None,
                                         "data": (tensor.handle.data_ptr(), False), "version": 2}


def _seen(tensor):
    t = torch.as_tensor(_Device(tensor), device="cuda")
    return t.view(torch.bfloat16) if tensor.dtype == "bfloat16" else t


def _framework():
    import kandle_amd

    try:
        kandle_amd.env.get_backend("hip")
    except RuntimeError:
        kandle_amd.HipBackend.create(0)
    return kandle_amd


def _put(x):
    """A framework tensor with x's values."""
    t = _framework().Tensor(shape=tuple(x.shape), dtype=_NAME[x.dtype])
    _seen(t).copy_(x)
    return t


def _results(case, x):
    """The framework tensors that a program lets the calls write to, by name (state they update included)."""
    new = lambda shape, dtype="int32": _framework().Tensor(shape=tuple(shape), dtype=dtype)  # noqa: E731
    kind = case["kind"]
    if kind == "attention":
        return {"o": new(x["q"].shape, case["dtype"])}
    if kind == "write":
        return {"kp": x["kp"], "vp": x["vp"]}
    if kind in ("step", "compact"):
        out = {"table": new(x["table"].shape), "refs": new(x["refs"].shape), "pages": x["pages"]}
        if kind == "step":
            return {**out, "lens": new(x["lens"].shape), "moves": new((x["lens"].shape[0], 2)), "info": new((3,))}
        return {**out, "moves": new((max(1, case["pages"] // 2), 2)), "info": new((2,))}
    shape = (case["groups"], case["beams"])
    out = {"scores": new(shape, "float32"), "tokens": new(shape), "parents": new(shape)}
    return {**out, "finished": new(shape)} if case["finished"] else out


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if own:  # the same values in the framework's own tensors, and its results as torch sees them
        state["x"] = {name: _put(v) for name, v in x.items()}
        state["out"] = _results(case, state["x"])
        state["seen"] = {name: _seen(v) for name, v in state["out"].items()}
    torch.cuda.synchronize()
    return state


def run(state):
    case, x, kind = state["case"], state["x"], state["case"]["kind"]
    if own:
        from kandle_amd import functional as F

        out = state["out"]
        if kind == "attention":
            F.paged_attention(x["q"], x["kp"], x["vp"], x["table"], x["lens"], x.get("starts"), max_query_len=case["new"],
                              max_kv_len=case["len"], out=out["o"])
            return state["seen"]["o"]
        if kind == "write":
            F.paged_kv_write(x["k"], x["v"], x["kp"], x["vp"], x["table"], x["lens"], x.get("starts"))
        elif kind == "step":
            F.pages_fork(x["table"], x["lens"], x["refs"], x["parents"], out=(out["table"], out["lens"], out["refs"]))
            F.pages_reserve(out["table"], out["lens"], out["refs"], x["counts"], case["page"], out=(out["moves"], out["info"]))
            F.pages_copy(x["pages"], out["moves"], out["info"])
        elif kind == "compact":
            F.pages_compact(x["table"], x["refs"], out=(out["table"], out["refs"], out["moves"], out["info"]))
            F.pages_copy(x["pages"], out["moves"], out["info"])
        else:
            F.beam_select(x["logits"], x["scores"], finished=x.get("finished"), eos_token_id=EOS,
                          out=(out["scores"], out["tokens"], out["parents"], out.get("finished")))
        return state["seen"]
    if kind == "attention":
        return _plain_attention(x, case)
    if kind == "write":
        return _plain_write(x, case)
    if kind == "step":
        return _plain_step(x, case)
    if kind == "compact":
        return _plain_compact(x, case)
    return _plain_select(x, case)


# ---------------------------------------------------------------------------------------------
# work / exact
# ---------------------------------------------------------------------------------------------
def work(case):
    size, kind = (2 if case["dtype"] == "bfloat16" else 4), case["kind"]
    if kind in ("attention", "write"):
        n, lens, table, _ = _geometry(case, 1)
        tokens, row = int(n.sum()), case["hkv"] * case["d"] * size
        if kind == "write":
            return {"bytes": 4 * tokens * row, "flops": 0}
        page = case["page"]
        key = np.arange(table.shape[1] * page)
        held = np.repeat(table >= 0, page, axis=1) & (key[None] < lens[:, None])
        # rows of pages that sequences share are needed once
        ids = np.where(held, np.repeat(table, page, axis=1) * page + key % page, -1)
        before = np.concatenate([np.zeros((len(lens), 1), np.int64), np.cumsum(held, 1)], 1)
        pairs = sum(int(before[i, lens[i] - n[i] + 1:lens[i] + 1].sum()) for i in range(len(lens)))
        return {"bytes": 2 * (len(np.unique(ids)) - bool((ids < 0).any())) * row + 2 * tokens * case["hq"] * case["d"] * size,
                "flops": 4 * case["d"] * case["hq"] * pairs}
    if kind == "select":
        rows = case["groups"] * case["beams"] * (0.75 if case["finished"] else 1)  # a finished beam's logits are not needed
        return {"bytes": rows * case["vocab"] * size + 20 * rows, "flops": 3 * rows * case["vocab"]}
    whole = case["layers"] * 2 * case["hkv"] * case["page"] * case["d"] * size
    if kind == "step":
        table, lens, refs, parents, pool = _beam_pages(case, 1)
        at, children = np.unique(parents, return_counts=True)
        copied = int(((children - 1) * (lens[at] % case["page"] != 0)).sum())  # all but one child of each parent
        return {"bytes": 2 * copied * whole + 8 * table.size + 8 * pool, "flops": 0}
    table, refs = _fragments(case, 1)
    live = int((refs > 0).sum())
    return {"bytes": 2 * int((refs[live:] > 0).sum()) * whole + 8 * table.size + 8 * len(refs), "flops": 0}


def exact(case, seed):
    x, kind = _inputs(case, seed), case["kind"]
    if kind == "attention":
        n, lens, table, _ = _geometry(case, seed)
        page, ratio, out, at = case["page"], case["hq"] // case["hkv"], [], 0
        for i in range(case["batch"]):
            rows = np.arange(lens[i])
            rows = rows[table[i, rows // page] >= 0]
            ids, slot = torch.from_numpy(table[i, rows // page]).cuda(), torch.from_numpy(rows % page).cuda()
            k, v = x["kp"][ids, :, slot].double(), x["vp"][ids, :, slot].double()  # [rows, hkv, d]
            q = x["q"][at:at + n[i]].double()
            at += n[i]
            hidden = torch.from_numpy(rows[None] > (lens[i] - n[i] + np.arange(n[i]))[:, None]).cuda()
            o = torch.zeros_like(q)
            if len(rows):
                for h in range(case["hq"]):
                    s = (q[:, h] @ k[:, h // ratio].t().contiguous()) / math.sqrt(case["d"])
                    o[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0) @ v[:, h // ratio].contiguous()
            out.append(o)
        return torch.cat(out)
    if kind == "select":
        logits, scores = x["logits"].cpu().double().numpy(), x["scores"].cpu().double().numpy()
        best = []
        for g in range(case["groups"]):
            every = []
            for b in range(case["beams"]):
                row = logits[g, b]
                if case["finished"] and int(x["finished"][g, b]):
                    every.append(np.array([scores[g, b]]))
                    continue
                top = row.max()
                got = row - (top + math.log(np.exp(row - top).sum())) + scores[g, b]
                every.append(np.partition(got, -case["beams"])[-case["beams"]:])
            best.append(np.sort(np.concatenate(every))[::-1][:case["beams"]])
        out = {"scores": torch.from_numpy(np.stack(best).copy()), "tokens": None, "parents": None}
        return {**out, "finished": None} if case["finished"] else out
    if kind == "write":
        n, lens, table, _ = _geometry(case, seed)
        page, at = case["page"], 0
        out = {"kp": x["kp"].double(), "vp": x["vp"].double()}
        for i in range(case["batch"]):
            rows = np.arange(lens[i] - n[i], lens[i])
            ids, slot = torch.from_numpy(table[i, rows // page]).cuda(), torch.from_numpy(rows % page).cuda()
            out["kp"][ids, :, slot] = x["k"][at:at + n[i]].double()
            out["vp"][ids, :, slot] = x["v"][at:at + n[i]].double()
            at += n[i]
        return out
    pages = x["pages"].double()
    if kind == "step":  # one row after another
        table, lens, refs, parents, _ = _beam_pages(case, seed)
        page, old = case["page"], table.copy()
        for i, parent in enumerate(parents):
            refs[old[i][old[i] >= 0]] -= 1
            table[i] = old[parent]
        for row in table:
            refs[row[row >= 0]] += 1
        lens, src, dst = lens[parents], [], []
        for i in range(len(table)):
            at, inside = divmod(int(lens[i]), page)
            if not inside or refs[table[i, at]] > 1:
                new = int(np.flatnonzero(refs == 0)[0])
                if inside:
                    src.append(int(table[i, at]))
                    dst.append(new)
                    refs[src[-1]] -= 1
                table[i, at], refs[new] = new, 1
        moves, info = np.full((len(table), 2), -1), [len(src), 0, 0]
        out = {"lens": torch.from_numpy(lens + 1)}
    else:
        table, refs = _fragments(case, seed)
        live = np.flatnonzero(refs)
        src = live[live >= len(live)]
        dst = np.setdiff1d(np.arange(len(live)), live)
        moves, info, out = np.full((max(1, case["pages"] // 2), 2), -1), [len(src), len(live)], {}
        for a, b in zip(src, dst):
            table[table == a], refs[b], refs[a] = b, refs[a], 0
    for i, (a, b) in enumerate(zip(src, dst)):
        moves[i] = a, b
        pages[:, :, b] = pages[:, :, a]
    return {**out, "table": torch.from_numpy(table), "refs": torch.from_numpy(refs), "moves": torch.from_numpy(moves),
            "info": torch.tensor(info), "pages": pages}
