"""Performance cases of the 8-bit paged KV cache: the append that rotates and
quantises, decode attention and packed prompt attention over the cache.

The cache. A block of `bs` tokens is one record per layer and K/V tensor: int8
codes of every KV head, then one f32 scale for each (head, token), padded to
256 bytes. K codes lie [head][token][dim], V codes [head][dim][token]. A row x
(one token of one head, K after its rotation) is held as

    scale = f32(max |x| / 127),   code = round(x / scale)   (ties to even)

and stands for code * scale.

A case is one of three kinds of work on one layer:

append   q and k rotated by their tokens' positions (angle = position * the
         pair's frequency), k and v quantised into their slots. Returns the
         rotated q and the cache's codes and scales.
decode   one query token per sequence over its whole cached context.
prefill  the query rows of several prompts of different lengths, packed one
         behind the other, each causal over its own cached context.

The attention shapes are those of rvllm_amd.workloads.CONFIGS, and head
dimensions between them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

#: name -> (query heads, KV heads, head_dim, block size)
SHAPES = {
    "smollm2-360m": (15, 5, 64, 16),
    "llama-3.2-1b": (32, 8, 64, 16),
    "qwen3-0.6b": (16, 8, 128, 16),
    "qwen2.5-0.5b": (14, 2, 64, 32),
    "gemma-3-270m": (4, 1, 256, 16),
    "odd-80": (12, 4, 80, 48),
    "odd-192": (9, 3, 192, 16),
    "wide-group": (22, 2, 128, 64),
}
DEV = "cuda"
F = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One step of eight chats: the smallest append, all latency.
        dict(name="append_step", kind="append", shape="qwen3-0.6b",
             dtype="f16", rows=8, rot=128, interleaved=False, far=4000,
             factor=1.0, norm=False),
        # Prompts of a serving batch, packed; K normed per head, as this shape
        # has it.
        dict(name="append_prompts", kind="append", shape="qwen3-0.6b",
             dtype="f16", rows=8191, rot=128, interleaved=False, far=40000,
             factor=1.0, norm=True),
        # A follow-up deep in a long document: interleaved pairs, half of each
        # head, positions near a million, the factor that scaled frequencies
        # come with.
        dict(name="append_far_partial", kind="append", shape="smollm2-360m",
             dtype="f32", rows=1999, rot=32, interleaved=True, far=1000000,
             factor=1.2079, norm=False),
        # One short chat: the smallest decode.
        dict(name="decode_one", kind="decode", shape="llama-3.2-1b",
             dtype="f16", batch=1, ctx=77, spread="uniform", window=0),
        # Two long documents, one user each: the context is split.
        dict(name="decode_long", kind="decode", shape="qwen3-0.6b",
             dtype="f32", batch=2, ctx=32749, spread="uniform", window=0),
        # The benchmark's headline batch.
        dict(name="decode_batch", kind="decode", shape="qwen3-0.6b",
             dtype="f16", batch=256, ctx=4096, spread="uniform", window=0),
        # A serving mix of contexts from 32 to 8192 tokens, seven heads a group.
        dict(name="decode_ragged", kind="decode", shape="qwen2.5-0.5b",
             dtype="f32", batch=512, ctx=8192, spread="log", window=0),
        # Sliding-window layers with a single KV head.
        dict(name="decode_window", kind="decode", shape="gemma-3-270m",
             dtype="f16", batch=96, ctx=5000, spread="log", window=512),
        # A few short prompts just admitted: the smallest packed call.
        dict(name="prefill_short", kind="prefill", shape="smollm2-360m",
             dtype="f16", seqs=5, q_len=61, offset=0, window=0),
        # Whole prompts of a serving batch, packed.
        dict(name="prefill_prompts", kind="prefill", shape="qwen3-0.6b",
             dtype="f16", seqs=7, q_len=4001, offset=0, window=0),
        # Chunks behind long cached contexts, in the f32 of the engine.
        dict(name="prefill_chunk", kind="prefill", shape="llama-3.2-1b",
             dtype="f32", seqs=2, q_len=300, offset=7700, window=0),
        # Prompts on sliding-window layers with a single KV head.
        dict(name="prefill_window", kind="prefill", shape="gemma-3-270m",
             dtype="f16", seqs=3, q_len=1500, offset=0, window=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    shape = rng.choice(sorted(SHAPES))
    H, kv, hd, _ = SHAPES[shape]
    c = dict(kind=kind, shape=shape, dtype=rng.choice(["f16", "f16", "f32"]))
    if kind == "append":
        c.update(rows=_log_int(rng, 1, 8000),
                 rot=rng.choice([hd, hd, hd // 2, hd // 4]),
                 interleaved=rng.random() < 0.4,
                 far=_log_int(rng, 9000, 2000000),
                 factor=rng.choice([1.0, round(rng.uniform(1.0, 1.5), 4)]),
                 norm=rng.random() < 0.4)
        return c
    while True:
        if kind == "decode":
            d = dict(c, batch=_log_int(rng, 1, 600),
                     ctx=_log_int(rng, 1, 40000),
                     spread=rng.choice(["uniform", "log"]),
                     window=rng.choice([0, 0, _log_int(rng, 16, 2000)]))
            # (the padded form's size too: short rows behind one long one)
            if work(d)["bytes"] <= 1e9 and d["batch"] * d["ctx"] * kv * hd <= 1e9:
                return d
        else:
            d = dict(c, seqs=rng.randint(1, 9), q_len=_log_int(rng, 1, 4000),
                     offset=rng.choice([0, 0, _log_int(rng, 5, 9000)]),
                     window=rng.choice([0, 0, _log_int(rng, 16, 2000)]))
            pairs = d["seqs"] * d["q_len"] * (d["offset"] + d["q_len"])
            if work(d)["flops"] <= 1.2e11 and pairs * H <= 1.5e9:
                return d


def _lens(case):
    """Each sequence's length, a function of the case alone (so that the
    work of a case is known without its inputs)."""
    if case["kind"] == "decode":
        n, top = case["batch"], case["ctx"]
        if case["spread"] == "uniform":
            return [top] * n
        lo = min(32, top)
        return [int(round(lo * (top / lo) ** ((i * 7919 % n) / max(1, n - 1))))
                for i in range(n)]
    n, top = case["seqs"], case["q_len"]
    order = [*range(0, n, 2), *range(1, n, 2)]
    return [max(1, top * (n - i) // n) for i in order]


def _rec(kv, hd, bs):
    return -(-kv * bs * (hd + 4) // 256) * 256


def _views(mem, which, nb, kv, hd, bs):
    """codes [nb, kv, bs, hd] int8 and scales [nb, kv, bs] f32 of a tensor."""
    rec = _rec(kv, hd, bs)
    row, dim = (hd, 1) if which == 0 else (1, bs)
    codes = mem.view(torch.int8).as_strided(
        (nb, kv, bs, hd), (rec, bs * hd, row, dim), which * nb * rec)
    scales = mem.view(torch.float32).as_strided(
        (nb, kv, bs), (rec // 4, bs, 1),
        (which * nb * rec + kv * bs * hd) // 4)
    return codes, scales


def _u32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int64)).to(DEV).to(
        torch.int32)


def _store(case, mem, nb):
    if not own:
        return None
    from rvllm_amd.q8_storage import HipQ8Storage
    _, kv, hd, bs = SHAPES[case["shape"]]
    return HipQ8Storage(1, nb, bs, kv, hd, memory=mem)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    H, kv, hd, bs = SHAPES[case["shape"]]
    dt = F[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "append":
        rows = case["rows"]
        # Sequences one behind the other, each at its own position, in blocks
        # of their own that lie anywhere in the pool.
        n_seq = min(rows, 8)
        cuts = [rows * i // n_seq for i in range(n_seq + 1)]
        lens = [b - a for a, b in zip(cuts, cuts[1:])]
        first = rng.integers(0, max(1, case["far"] - max(lens)), n_seq)
        pos = np.concatenate([f + np.arange(n) for f, n in zip(first, lens)])
        need = [-(-(f % bs + n) // bs) for f, n in zip(first, lens)]
        nb = sum((n + 2 * bs - 2) // bs for n in lens)  # (whatever the starts)
        ids, at, blk = rng.permutation(nb), 0, []
        for f, n, k in zip(first, lens, need):
            blk.append(ids[at + (f % bs + np.arange(n)) // bs])
            at += k
        qkv = torch.randn((rows, (H + 2 * kv) * hd), generator=g, device=DEV)
        # (a few large channels, as keys have them)
        amp = torch.exp2(2 * torch.randn(((H + 2 * kv) * hd,), generator=g,
                                         device=DEV).clamp(-1.5, 1.5))
        qkv = (qkv * amp).to(dt)
        split = [H * hd, kv * hd, kv * hd]
        q, k, v = (t.view(rows, -1, hd) for t in qkv.split(split, dim=1))
        rot = case["rot"]
        inv = (1e6 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)
        mem = torch.zeros(2 * nb * _rec(kv, hd, bs), dtype=torch.uint8,
                          device=DEV)
        w = [1 + 0.1 * torch.randn(hd, generator=g, device=DEV)
             for _ in range(2)] if case["norm"] else [None, None]
        s.update(q=q, k=k, v=v, pos=_u32(pos), inv=torch.from_numpy(inv).to(
            DEV), blk=_u32(np.concatenate(blk)), off=_u32(pos % bs), mem=mem,
            nb=nb, q_norm=w[0], k_norm=w[1], store=_store(case, mem, nb))
        return s
    lens = _lens(case)
    off = case.get("offset", 0)
    ctx = lens if case["kind"] == "decode" else [off + n for n in lens]
    need = [-(-n // bs) for n in ctx]
    nb = sum(need)
    ids, at = rng.permutation(nb), np.concatenate([[0], np.cumsum(need)])
    wide = max(need)
    tables = np.stack([ids[np.minimum(a + np.arange(wide), a + k - 1)]
                       for a, k in zip(at, need)])
    mem = torch.zeros(2 * nb * _rec(kv, hd, bs), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (kv * bs * hd))
    for which in (0, 1):
        codes, scales = _views(mem, which, nb, kv, hd, bs)
        for a in range(0, nb, step):
            n = min(step, nb - a)
            x = torch.randn((n, kv, bs, hd), generator=g, device=DEV)
            x *= torch.exp2(torch.randn((n, kv, bs, 1), generator=g,
                                        device=DEV) * 0.5)
            sc = x.abs().amax(-1) / 127
            scales[a:a + n] = sc
            codes[a:a + n] = torch.round(x / sc[..., None]).to(torch.int8)
    rows = len(lens) if case["kind"] == "decode" else sum(lens)
    s.update(q=torch.randn((rows, H, hd), generator=g, device=DEV).to(dt),
             tables=_u32(tables), reads=_u32(ctx), mem=mem, nb=nb,
             wide=max(ctx), store=_store(case, mem, nb))
    if case["kind"] == "prefill":
        s.update(starts=_u32(np.concatenate([[0], np.cumsum(lens)])),
                 offs=_u32([off] * len(lens)), q_max=max(lens))
    elif own:
        s["ws"] = s["store"].alloc_workspace(len(lens), H, max(ctx))
    return s


def run(s):
    c = s["case"]
    if not own:
        return _plain[c["kind"]](s)
    st = s["store"]
    if c["kind"] == "append":
        q = st.rope_append(0, s["q"], s["k"], s["v"], s["pos"], s["inv"],
                           s["blk"], s["off"], interleaved=c["interleaved"],
                           attn_factor=c["factor"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=1e-6)
        return dict(q=q, k_codes=st.codes(0, 0), k_scales=st.scales(0, 0),
                    v_codes=st.codes(0, 1), v_scales=st.scales(0, 1))
    if c["kind"] == "decode":
        return st.paged_decode(0, s["q"], s["tables"], s["reads"], s["wide"],
                               ws=s["ws"], window=c["window"])
    return st.packed_prefill(0, s["q"], s["starts"], s["tables"], s["offs"],
                             s["reads"], window=c["window"])


# -- the plain forms ----------------------------------------------------------

def _rotate(x, cos, sin, rot, interleaved):
    """x [rows, heads, hd] f64; cos, sin [rows, 1, rot / 2]."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
    u, v = a * cos - b * sin, a * sin + b * cos
    r = (torch.stack([u, v], -1).flatten(-2) if interleaved
         else torch.cat([u, v], -1))
    return torch.cat([r, rest], -1)


def _quantise(x):
    scale = (x.abs().amax(-1) / 127).to(torch.float32)
    code = torch.round(x / scale.double()[..., None]).clamp(-127, 127)
    return torch.where(scale[..., None] > 0, code, 0).to(torch.int8), scale


def _plain_append(s):
    # In 64 bits: angles of far positions, values next to a code's border.
    c = s["case"]
    _, kv, hd, bs = SHAPES[c["shape"]]
    ang = s["pos"].double()[:, None] * s["inv"].double()
    cos, sin = ((f(ang) * c["factor"])[:, None] for f in (torch.cos,
                                                          torch.sin))
    q, k, v = (s[n].double() for n in "qkv")
    if c["norm"]:
        q, k = (x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
                * s[w].double() for x, w in ((q, "q_norm"), (k, "k_norm")))
    q = _rotate(q, cos, sin, c["rot"], c["interleaved"]).to(s["q"].dtype)
    k = _rotate(k, cos, sin, c["rot"], c["interleaved"])
    blk, off = s["blk"].long(), s["off"].long()
    out = dict(q=q)
    for which, name, x in ((0, "k", k), (1, "v", v)):
        codes, scales = _views(s["mem"], which, s["nb"], kv, hd, bs)
        codes[blk, :, off], scales[blk, :, off] = _quantise(x)
        out[name + "_codes"], out[name + "_scales"] = codes, scales
    return out


def _dense(s):
    """Every sequence's K and V in f32, [batch, kv, tokens, hd]."""
    _, kv, hd, bs = SHAPES[s["case"]["shape"]]
    at = s["tables"].long()
    got = []
    for which in (0, 1):
        codes, scales = _views(s["mem"], which, s["nb"], kv, hd, bs)
        x = codes[at].float() * scales[at][..., None]
        got.append(x.transpose(1, 2).reshape(at.shape[0], kv, -1, hd))
    return got


def _attend(q, k, v, seen):
    """q [b, kv, rows, hd], seen [b, 1, rows, tokens]: softmax(q k') v."""
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(q.shape[-1])
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    w = torch.exp(x - top)
    return torch.matmul(w, v) / w.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_decode(s):
    c = s["case"]
    H, kv, hd, _ = SHAPES[c["shape"]]
    k, v = _dense(s)
    j = torch.arange(k.shape[2], device=DEV)[None]
    n = s["reads"].long()[:, None]
    seen = j < n
    if c["window"]:
        seen = seen & (j + c["window"] > n - 1)
    q = s["q"].float().view(-1, kv, H // kv, hd)
    return _attend(q, k, v, seen[:, None, None]).reshape(
        -1, H, hd).to(s["q"].dtype)


def _plain_prefill(s):
    # The packed rows spread out to [batch, longest], and back.
    c = s["case"]
    H, kv, hd, _ = SHAPES[c["shape"]]
    k, v = _dense(s)
    starts = s["starts"].long()
    rows = s["q"].shape[0]
    at = torch.arange(rows, device=DEV)
    b = torch.searchsorted(starts, at, right=True) - 1
    i = at - starts[b]
    q = torch.zeros((starts.numel() - 1, s["q_max"], H, hd), device=DEV)
    q[b, i] = s["q"].float()
    G = H // kv
    q = q.view(q.shape[0], s["q_max"], kv, G, hd).permute(0, 2, 3, 1, 4)
    pos = s["offs"].long()[:, None] + torch.arange(s["q_max"], device=DEV)
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= pos[..., None]) & (j < s["reads"].long()[:, None, None])
    if c["window"]:
        seen = seen & (j + c["window"] > pos[..., None])
    seen = seen[:, None, None].expand(-1, -1, G, -1, -1).flatten(2, 3)
    o = _attend(q.flatten(2, 3), k, v, seen)
    o = o.view(o.shape[0], kv, G, s["q_max"], hd).permute(0, 3, 1, 2, 4)
    return o[b, i].reshape(rows, H, hd).to(s["q"].dtype)


_plain = dict(append=_plain_append, decode=_plain_decode,
              prefill=_plain_prefill)


# -- what a pass cannot do without --------------------------------------------

def work(case):
    H, kv, hd, bs = SHAPES[case["shape"]]
    eb = 2 if case["dtype"] == "f16" else 4
    if case["kind"] == "append":
        rows = case["rows"]
        n = rows * (H + 2 * kv) * hd
        cell = rows * 2 * kv * (hd + 4)
        return dict(bytes=n * eb + rows * H * hd * eb + cell + rows * 12
                    + case["rot"] * 2, flops=8 * n)
    lens, win = _lens(case), case["window"]
    if case["kind"] == "decode":
        seen = [min(n, win) if win else n for n in lens]
        keys, pairs, rows = sum(seen), sum(seen), len(lens)
    else:
        off, rows, pairs, keys = case["offset"], sum(lens), 0, 0
        for n in lens:
            if not win:
                pairs += n * off + n * (n + 1) // 2
                keys += off + n
                continue
            grow = min(n, max(0, win - off))  # rows that see less than win
            pairs += grow * off + grow * (grow + 1) // 2 + (n - grow) * win
            keys += min(off, win - 1) + n
    return dict(bytes=keys * kv * 2 * (hd + 4) + 2 * rows * H * hd * eb
                + 4 * (-(-keys // bs) + 3 * len(lens)),
                flops=4 * pairs * H * hd)


# -- the definition in 64 bits ------------------------------------------------

def _cells(s, which, blocks):
    """What the listed blocks' cells stand for, f64 [tokens, kv, hd], read
    from the records byte by byte's place."""
    _, kv, hd, bs = SHAPES[s["case"]["shape"]]
    rec = _rec(kv, hd, bs)
    raw = s["mem"].view(-1, rec)[which * s["nb"] + blocks]
    n = kv * bs * hd
    code = raw[:, :n].contiguous().view(torch.int8).double()
    scale = raw[:, n:n + 4 * kv * bs].contiguous().view(torch.float32)
    code = (code.view(-1, kv, bs, hd) if which == 0
            else code.view(-1, kv, hd, bs).transpose(2, 3))
    x = code * scale.double().view(-1, kv, bs, 1)
    return x.transpose(1, 2).reshape(-1, kv, hd)


def exact(case, seed):
    s = prepare(case, seed)
    H, kv, hd, bs = SHAPES[case["shape"]]
    if case["kind"] == "append":
        ang = torch.outer(s["pos"].double(), s["inv"].double())
        turn = torch.polar(torch.full_like(ang, case["factor"]), ang)[:, None]
        half = case["rot"] // 2
        first = (torch.arange(half, device=DEV) * 2 if case["interleaved"]
                 else torch.arange(half, device=DEV))
        second = first + (1 if case["interleaved"] else half)

        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + 1e-6)
                x = x * w.double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        k, v = turned(s["k"], s["k_norm"]), s["v"].double()
        out = dict(q=turned(s["q"], s["q_norm"]), k_codes=None, v_codes=None)
        for name, x in (("k", k), ("v", v)):
            sc = torch.zeros((s["nb"], kv, bs), dtype=torch.float64,
                             device=DEV)
            sc[s["blk"].long(), :, s["off"].long()] = \
                x.abs().max(-1).values / 127
            out[name + "_scales"] = sc
        return out
    lens, win = _lens(case), case["window"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    row = 0
    for b, n in enumerate(lens):
        total = int(s["reads"][b])
        blocks = s["tables"][b, :-(-total // bs)].long()
        k, v = (_cells(s, which, blocks)[:total] for which in (0, 1))
        m = 1 if case["kind"] == "decode" else n
        pos = total - m + torch.arange(m, device=DEV)
        j = torch.arange(total, device=DEV)
        hide = j > pos[:, None]
        if win:
            hide = hide | (j <= pos[:, None] - win)
        for h in range(H):
            a = q[row:row + m, h] @ k[:, h * kv // H].T * hd ** -0.5
            a = torch.where(hide, -math.inf, a)
            a = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
            out[row:row + m, h] = a @ v[:, h * kv // H]
        row += m
    return out
