"""The operators of the paged key-value cache, as cases that can be timed and checked.

A case is a dict of plain values: `kind` names the operator (append: new keys and values into
the cache's pages with the rotation on the way; decode: attention of one new token of every
sequence; prompt: attention of several new tokens of every sequence), the rest its sizes and
options.  listed() gives the standing ones, draw() more of the same ranges.

With `own` false run() computes the operator in plain torch, in 32 bits, rounded once at the
end; with `own` true it calls the framework.  exact() is the same from the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

# Head geometries (query heads, kv heads, head_dim) and RoPE bases of the benchmark's decode and
# prompt workloads ("8b", "4b"), and of the decode tests.
SHAPES = {
    "8b": (32, 8, 128, 500000.0),
    "4b": (8, 4, 256, 10000.0),
    "mha64": (8, 8, 64, 10000.0),
    "gqa96": (24, 8, 96, 10000.0),
    "gqa64": (8, 2, 64, 500000.0),
    "mqa256": (4, 1, 256, 10000.0),
}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0


def listed():
    return [
        # one chat's next token: the smallest call, launch and latency
        {"name": "append_1", "kind": "append", "shape": "8b", "act": "f32", "kv": "f16", "page": 16, "layout": "token",
         "seqs": 1, "new": 1, "old": 2048, "rotary": 0},
        # seven users' prompts of different lengths at once, some continuing a conversation
        {"name": "append_prompts", "kind": "append", "shape": "8b", "act": "f32", "kv": "f16", "page": 16,
         "layout": "head", "seqs": 7, "new": 1100, "old": 300, "rotary": 0},
        # a long document into an 8-bit cache, half of each head rotated
        {"name": "append_e4m3", "kind": "append", "shape": "4b", "act": "bf16", "kv": "e4m3", "page": 64,
         "layout": "head", "seqs": 1, "new": 8191, "old": 0, "rotary": 128},
        # one chat's next token over a short history
        {"name": "decode_1_short", "kind": "decode", "shape": "8b", "act": "f32", "kv": "f16", "page": 16,
         "layout": "token", "seqs": 1, "len": 517, "ragged": False, "window": 0, "softcap": 0.0},
        # a server's step: 32 users with histories of every length
        {"name": "decode_32", "kind": "decode", "shape": "8b", "act": "f32", "kv": "f16", "page": 16, "layout": "head",
         "seqs": 32, "len": 4096, "ragged": True, "window": 0, "softcap": 0.0},
        # one user with a book in the context
        {"name": "decode_1_long", "kind": "decode", "shape": "8b", "act": "bf16", "kv": "bf16", "page": 64,
         "layout": "head", "seqs": 1, "len": 131071, "ragged": False, "window": 0, "softcap": 0.0},
        # a full server on an 8-bit cache
        {"name": "decode_64_e4m3", "kind": "decode", "shape": "8b", "act": "bf16", "kv": "e4m3", "page": 32,
         "layout": "head", "seqs": 64, "len": 12000, "ragged": True, "window": 0, "softcap": 0.0},
        # the sliding-window layers with capped scores
        {"name": "decode_window", "kind": "decode", "shape": "4b", "act": "f32", "kv": "f16", "page": 256,
         "layout": "token", "seqs": 48, "len": 6000, "ragged": True, "window": 1024, "softcap": 50.0},
        # the benchmark's 512-token prompt
        {"name": "prompt_512", "kind": "prompt", "shape": "8b", "act": "f32", "kv": "f16", "page": 16,
         "layout": "head", "seqs": 1, "new": 512, "old": 0, "window": 0, "softcap": 0.0},
        # drafted tokens of eight users checked against long histories
        {"name": "prompt_drafts", "kind": "prompt", "shape": "8b", "act": "bf16", "kv": "e4m3", "page": 32,
         "layout": "head", "seqs": 8, "new": 9, "old": 15000, "window": 0, "softcap": 0.0},
        # chunks of several users' prompts behind what is already cached
        {"name": "prompt_chunks", "kind": "prompt", "shape": "8b", "act": "bf16", "kv": "bf16", "page": 16,
         "layout": "token", "seqs": 5, "new": 1200, "old": 2500, "window": 0, "softcap": 0.0},
        # a long document at once
        {"name": "prompt_8k", "kind": "prompt", "shape": "8b", "act": "bf16", "kv": "bf16", "page": 64,
         "layout": "head", "seqs": 1, "new": 8191, "old": 0, "window": 0, "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    act, kv = rng.choice([("f32", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "e4m3"), ("f16", "f16"),
                          ("bf16", "bf16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")])
    shape = rng.choice(["8b", "8b", "8b", "4b", "4b", "mha64", "gqa96", "gqa64", "mqa256"])
    c = {"kind": kind, "shape": shape, "act": act, "kv": kv, "page": rng.choice([16, 16, 32, 64, 128, 256, 1, 8, 40]),
         "layout": rng.choice(["token", "head"])}
    seqs = _log(rng, 1, 64)
    if kind == "append":  # one token of each sequence, or prompts
        hd = SHAPES[shape][2]
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 8000 // seqs))
        return c | {"seqs": seqs, "new": new, "old": _log(rng, 1, max(2, 9000 // seqs)),
                    "rotary": rng.choice([0, 0, hd // 2, 32])}
    window = rng.choice([0, 0, 0, 1024, _log(rng, 1, 4000)])
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0, 50.0])
    if kind == "decode":
        return c | {"seqs": seqs, "len": _log(rng, 1, min(131072, 200000 // seqs)), "ragged": rng.random() < 0.7,
                    "window": window, "softcap": softcap}
    seqs = _log(rng, 1, 16)
    new = _log(rng, 2, max(2, 6000 // seqs))
    return c | {"seqs": seqs, "new": new, "old": _log(rng, 1, min(16000, 40000 // seqs, max(2, 12000000 // (seqs * new)))),
                "window": window, "softcap": softcap}


# ── sizes of a case ────────────────────────────────────────────────────────
def _lengths(c):
    """(new tokens, cached positions with them) of every sequence: ragged, the same for every seed."""
    n = c["seqs"]
    if c["kind"] == "decode":
        lens = [max(1, c["len"] * (1 + 37 * i % n) // n) if c["ragged"] else c["len"] for i in range(n)]
        return [1] * n, lens
    new = [c["new"] if i == 0 or c["new"] == 1 else max(1, c["new"] * (1 + (11 * i) % n) // n) for i in range(n)]
    old = [c["old"] * ((13 * i + n - 1) % n + 1) // n for i in range(n)]
    return new, [a + b for a, b in zip(new, old)]


def _keys(c, new, lens):
    """Positions that a sequence's new tokens read, and the (token, position) pairs of all of them."""
    w = c["window"] or 1 << 60
    read = pairs = 0
    for n, L in zip(new, lens):
        read += L - max(0, L - n + 1 - w)
        pairs += sum(min(w, L - n + 1 + i) for i in range(n))
    return read, pairs


def work(case):
    nq, nkv, hd, _ = SHAPES[case["shape"]]
    new, lens = _lengths(case)
    a, e, T = BYTES[case["act"]], BYTES[case["kv"]], sum(new)
    if case["kind"] == "append":
        return {"bytes": T * hd * ((nq + 2 * nkv) * a + nq * a + 2 * nkv * e), "flops": 6 * T * hd * (nq + nkv) // 2}
    read, pairs = _keys(case, new, lens)
    return {"bytes": 2 * read * nkv * hd * e + 2 * T * nq * hd * a, "flops": 4 * pairs * nq * hd}


# ── what a program holds before the call ───────────────────────────────────
def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _pages(gen, c, pages, nkv, hd, scale):
    """Pages of keys or values as [page][position][head][dim], in the case's memory order."""
    dims = (pages, c["page"], nkv, hd) if c["layout"] == "token" else (pages, nkv, c["page"], hd)
    t = torch.empty(dims, device="cuda", dtype=TYPES[c["kv"]])
    step = max(1, (64 << 20) // (dims[1] * dims[2] * dims[3]))
    for p in range(0, pages, step):  # bounded temporaries
        t[p:p + step] = _normal(gen, (min(step, pages - p),) + dims[1:], torch.float32, 1.0 / scale).to(TYPES[c["kv"]])
    return t if c["layout"] == "token" else t.transpose(1, 2)


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda").manual_seed(seed)
    nq, nkv, hd, base = SHAPES[c["shape"]]
    new, lens = _lengths(c)
    act, T, P = TYPES[c["act"]], sum(new), c["page"]
    need = [-(-L // P) for L in lens]
    width, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    start = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32)
    s = {"case": c, "nq": nq, "nkv": nkv, "hd": hd, "base": base, "max_new": max(new), "max_len": max(lens),
         "table": table.cuda(), "kv_len": torch.tensor(lens, dtype=torch.int32).cuda(),
         "q_start": None if c["kind"] == "decode" else start.cuda(), "tokens": T}
    scale = 1.0
    if c["kv"] == "e4m3":  # scales per kv head, near the largest value over e4m3's largest
        s["k_scale"] = 0.012 * (1 + torch.rand(nkv, generator=gen, device="cuda"))
        s["v_scale"] = 0.012 * (1 + torch.rand(nkv, generator=gen, device="cuda"))
        scale = 0.018
    s["k_pages"], s["v_pages"] = _pages(gen, c, pages, nkv, hd, scale), _pages(gen, c, pages, nkv, hd, scale)
    if c["kind"] == "append":  # one projection's rows [q | k | v], as the products write them
        s["qkv"] = _normal(gen, (T, (nq + 2 * nkv) * hd), act)
        s["out"] = torch.empty(T, nq, hd, device="cuda", dtype=act)
    else:
        s["q"] = _normal(gen, (T, nq, hd), act, 1.5)
        s["out"] = torch.empty(T, nq, hd, device="cuda", dtype=act)
    if own:
        be, larql_hip = _backend()
        s["be"] = be
        s["kv"] = larql_hip.PagedKV(s["k_pages"], s["v_pages"], s.get("k_scale"), s.get("v_scale"))
        s["batch"] = larql_hip.PagedBatch(s["table"], s["kv_len"], s["q_start"], tokens=T)
        s["stream"] = _stream()
        if c["kind"] != "append":
            n = be.paged_attention_work_bytes(s["kv"], s["batch"], nq)
            s["work"] = torch.empty(max(16, n), device="cuda", dtype=torch.uint8)
        s["stream"].wait_stream(torch.cuda.current_stream())  # what was made above
    return s


_be = None
_streams = []


def _stream():
    """The one stream of every pass, as in a serving loop."""
    if not _streams:
        _streams.append(torch.cuda.Stream())
    return _streams[0]


def _backend():
    global _be
    if _be is None:
        sys.path.insert(0, os.path.abspath("encoding-experiment_amd"))
        import larql_hip
        _be = larql_hip.HipBackend(0, strict=True), larql_hip
    return _be


# ── one pass ───────────────────────────────────────────────────────────────
def run(state):
    s, c = state, state["case"]
    if c["kind"] == "append":
        if own:
            nq, nkv, hd = s["nq"], s["nkv"], s["hd"]
            q, k, v = s["qkv"].split([nq * hd, nkv * hd, nkv * hd], dim=1)
            s["be"].paged_append_dev(s["kv"], s["batch"], k, v, q=q, q_out=s["out"], rope_base=s["base"],
                                     rotary_dim=c["rotary"], stream=s["stream"])
            return s["k_pages"], s["v_pages"], s["out"]
        return _plain_append(s)
    if own:
        s["be"].paged_attention_dev(s["kv"], s["batch"], s["q"], s["out"], scale=s["hd"] ** -0.5, window=c["window"],
                                    softcap=c["softcap"], work=s["work"], stream=s["stream"])
        return s["out"]
    return _plain_attention(s)


# ── the plain forms ────────────────────────────────────────────────────────
def _places(s):
    """Sequence, position and place among its sequence's new tokens of every token row."""
    rows = torch.arange(s["tokens"], device="cuda")
    if s["q_start"] is None:
        return rows, s["kv_len"].long() - 1, torch.zeros_like(rows)
    start = s["q_start"].long()
    seq = torch.searchsorted(start, rows, right=True) - 1
    i = rows - start[seq]
    return seq, s["kv_len"].long()[seq] - (start[seq + 1] - start[seq]) + i, i


def _plain_append(s):
    c, nq, nkv, hd, P = s["case"], s["nq"], s["nkv"], s["hd"], s["case"]["page"]
    seq, pos, _ = _places(s)
    x = s["qkv"].float().view(s["tokens"], nq + 2 * nkv, hd)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    half = (c["rotary"] or hd) // 2
    freq = torch.pow(torch.tensor(s["base"], device="cuda", dtype=torch.float64),
                     -torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = pos.double()[:, None, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, qk[..., 2 * half:]], -1)
    k, kv = qk[:, nq:], TYPES[c["kv"]]
    if c["kv"] == "e4m3":
        k = (k * (1.0 / s["k_scale"])[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        v = (v * (1.0 / s["v_scale"])[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    page, off = s["table"].long()[seq, pos // P], pos % P
    if c["kv"] == "e4m3":  # a byte view: 8-bit floating types are not written by index
        s["k_pages"].view(torch.uint8)[page, off] = k.to(kv).view(torch.uint8)
        s["v_pages"].view(torch.uint8)[page, off] = v.to(kv).view(torch.uint8)
    else:
        s["k_pages"][page, off] = k.to(kv)
        s["v_pages"][page, off] = v.to(kv)
    s["out"].copy_(qk[:, :nq])
    return s["k_pages"], s["v_pages"], s["out"]


def _gather(pages, table, pos, P, scale):
    """[sequence][position][head][dim] in f32 of the positions 0 .. max."""
    raw = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
    got = raw[table.long().clamp(min=0)[:, pos // P], pos % P]
    got = got.view(torch.float8_e4m3fn).float() if pages.dtype == torch.float8_e4m3fn else got.float()
    return got if scale is None else got * scale[:, None]


def _plain_attention(s):
    c, nq, nkv, hd, n = s["case"], s["nq"], s["nkv"], s["hd"], s["kv_len"].numel()
    seq, place, i = _places(s)
    pos = torch.arange(s["max_len"], device="cuda")
    k = _gather(s["k_pages"], s["table"], pos, c["page"], s.get("k_scale"))
    v = _gather(s["v_pages"], s["table"], pos, c["page"], s.get("v_scale"))
    q = torch.zeros(n, s["max_new"], nq, hd, device="cuda")
    q[seq, i] = s["q"].float()
    t = torch.full((n, s["max_new"]), -1, device="cuda")
    t[seq, i] = place
    seen = (pos <= t[..., None]) & (pos > t[..., None] - (c["window"] or 1 << 40))  # [seq][row][position]
    q = q.view(n, s["max_new"], nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * hd ** -0.5
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    x = x.view(n, nkv, nq // nkv, s["max_new"], -1).masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1)
    o = torch.matmul(p.view(n, nkv, -1, p.shape[-1]), v.transpose(1, 2).contiguous())
    o = o.view(*p.shape[:-1], hd) / total.clamp(min=1e-30)[..., None]  # [seq][kv][rep][row][dim]
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], nq, hd)[seq, i])
    return s["out"]


# ── from the definition, in 64 bits ────────────────────────────────────────
def _codes(t):
    return t.contiguous().double() if t.dtype != torch.float8_e4m3fn else t.contiguous().float().double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    nq, nkv, hd, base = SHAPES[c["shape"]]
    new, lens = _lengths(c)
    P, table = c["page"], s["table"].cpu()
    if c["kind"] == "append":
        K, V, out, at, r = _codes(s["k_pages"]), _codes(s["v_pages"]), [], 0, c["rotary"] or hd
        ks = s["k_scale"].double()[:, None] if "k_scale" in s else 1.0
        vs = s["v_scale"].double()[:, None] if "v_scale" in s else 1.0
        for b, (n, L) in enumerate(zip(new, lens)):
            x = s["qkv"][at:at + n].double().view(n, -1, hd)
            at += n
            t = torch.arange(L - n, L)
            ang = t.double()[:, None] * torch.tensor([base ** (-2.0 * j / r) for j in range(r // 2)], dtype=torch.float64)
            z = torch.polar(torch.ones_like(ang), ang).cuda()[:, None, :]
            w = torch.complex(x[..., :r // 2], x[..., r // 2:r])[:, :nq + nkv] * z
            x[:, :nq + nkv, :r // 2], x[:, :nq + nkv, r // 2:r] = w.real, w.imag
            out.append(x[:, :nq])
            page, off = table[b].long()[t // P].cuda(), (t % P).cuda()
            K[page, off], V[page, off] = x[:, nq:nq + nkv] / ks, x[:, nq + nkv:] / vs
        return K, V, torch.cat(out)
    if _keys(c, new, lens)[1] * nq * hd > 6e12:
        return None
    out, at = [], 0
    for b, (n, L) in enumerate(zip(new, lens)):
        t = torch.arange(L)
        page, off = table[b].long()[t // P].cuda(), (t % P).cuda()
        pos = torch.arange(L, device="cuda")
        me = torch.arange(L - n, L, device="cuda")[:, None]
        hide = (pos > me) | (pos <= me - (c["window"] or 1 << 40))
        o = torch.empty(n, nq, hd, device="cuda", dtype=torch.float64)
        for h in range(nkv):
            k, v = (_codes(s[x][:, :, h])[page, off] for x in ("k_pages", "v_pages"))
            if "k_scale" in s:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            for j in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                x = s["q"][at:at + n, j].double() @ k.T.contiguous() / math.sqrt(hd)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                x[hide] = float("-inf")
                o[:, j] = torch.softmax(x, 1) @ v
        at += n
        out.append(o)
    return torch.cat(out)
