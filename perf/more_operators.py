"""The operators of a cache that holds keys and values in 4 bits, as measured cases.

The cache's format is MXFP4: e2m1 codes with one power of two per 32 channels of a token, in 64-token pages.  Four
kinds of call, in the order of a model's layer:

  rotate    rotary positions with several axes (time, height, width) on queries and keys
  append    queries and keys rotated, keys and values quantised into the pages; what the cache then holds comes back
            as values: with the call itself, or read back from the pages together with the tokens before them
  readback  keys and values of whole sequences out of the pages, for attention that takes them dense
  attend    exact attention of the L newest tokens of every sequence over the pages

`run` computes them in plain torch operations, or, where `own` is true, by the framework's calls.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

D = 128
PAGE = 64
BLOCK = 32  # channels of a scale
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LOW, _HIGH, _NAN = 105, 140, 255  # scale bytes in use: 2^-22 .. 2^13


# ---------------------------------------------------------------------------- the cases
def _rotate(name, B, T, HQ, HKV, sections, dtype="bf16", pairs="half", order="blocks", inverse=False, far=0):
    return {"name": name, "kind": "rotate", "B": B, "T": T, "HQ": HQ, "HKV": HKV, "sections": sections, "dtype": dtype,
            "pairs": pairs, "order": order, "inverse": inverse, "far": far}


def _append(name, B, T, before, HQ, HKV, sections="", dtype="bf16", pairs="half", order="blocks"):
    return {"name": name, "kind": "append", "B": B, "T": T, "before": before, "HQ": HQ, "HKV": HKV,
            "sections": sections, "dtype": dtype, "pairs": pairs, "order": order}


def _readback(name, B, lo, hi, HKV, dtype="bf16"):
    return {"name": name, "kind": "readback", "B": B, "lo": lo, "hi": hi, "HKV": HKV, "dtype": dtype}


def _attend(name, B, L, lo, hi, HQ=32, HKV=8, dtype="bf16", padded=False):
    return {"name": name, "kind": "attend", "B": B, "L": L, "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV, "dtype": dtype,
            "padded": padded}


def listed():
    return [
        # one token of each of 64 sequences, far into long videos: latency
        _rotate("rotate_step_b64", 64, 1, 32, 8, "16,24,24", far=100000),
        # a video prompt of 16K tokens in time, height and width
        _rotate("rotate_video_16k", 1, 16384, 32, 8, "16,24,24"),
        # images in height and width, fp32, adjacent pairs, rotated back (the gradient of a prompt)
        _rotate("rotate_back_b3", 3, 701, 28, 4, "32,32", dtype="fp32", pairs="adjacent", inverse=True),
        # a decode step of 64 sequences: one token each, rotated and stored
        _append("append_step_b64", 64, 1, 4096, 32, 8, "24,20,20", order="cycled"),
        # a 16K-token prompt, rotated and stored; its attention takes the values as the cache holds them
        _append("append_prompt_16k", 1, 16384, 0, 32, 8, "16,24,24"),
        # chunks of five sequences at odd positions behind earlier tokens, stored as they are and read back whole
        _append("append_chunks_b5", 5, 333, 1001, 0, 4, dtype="fp16"),
        # one short sequence read back: latency
        _readback("readback_b1_2k", 1, 2000, 2000, 8),
        # four long ragged sequences read back
        _readback("readback_b4_32k", 4, 8192, 32768, 8),
        # one short conversation, one token: latency
        _attend("attend_b1_2k", 1, 1, 2000, 2000),
        # a serving batch of long, ragged contexts, one token each: the cache's bytes
        _attend("attend_b16_ragged", 16, 1, 8192, 65536),
        # five drafted tokens of each of eight sequences
        _attend("attend_draft_b8", 8, 5, 8192, 65536, dtype="fp16"),
        # the last 2K tokens of a 16K prompt: a chunk of a long prefill
        _attend("attend_chunk_2k_of_16k", 1, 2048, 16384, 16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "readback", "attend", "attend", "attend"])
    HKV = rng.choice([1, 2, 4, 8, 8])
    HQ = HKV * rng.choice([1, 2, 4, 4, 7, 8])
    axes = rng.choice([1, 2, 3, 3])
    a = rng.randint(8, 40)
    b = rng.randint(8, 56 - a)
    rope = {"sections": ["64", f"{a},{64 - a}", f"{a},{b},{64 - a - b}"][axes - 1], "pairs": rng.choice(["half", "half", "adjacent"]),
            "order": rng.choice(["blocks", "cycled"])}
    if kind == "rotate":
        B = _log(rng, 1, 64)
        T = max(1, min(_log(rng, 1, 16384), 16384 * 40 // (B * (HQ + HKV))))
        c = _rotate("", B, T, HQ, HKV, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), inverse=rng.random() < 0.3,
                    far=rng.choice([0, 0, 100000]), **rope)
        if c["dtype"] == "fp32":
            c["T"] = (c["T"] + 1) // 2
    elif kind == "append":
        B = _log(rng, 1, 128)
        T = rng.choice([1, _log(rng, 2, 64), _log(rng, 64, 16384)])
        T = max(1, min(T, 16384 // B))
        if rng.random() < 0.3:  # as it is, and read back
            c = _append("", B, T, _log(rng, 1, max(2, 8192 // B)), 0, HKV, dtype=rng.choice(["bf16", "fp16"]))
        else:
            c = _append("", B, T, _log(rng, 1, 4096), HQ, HKV, dtype=rng.choice(["bf16", "fp16"]), **rope)
    elif kind == "readback":
        hi = _log(rng, 1, 32768)
        B = max(1, min(_log(rng, 1, 32), 80000 // hi))
        c = _readback("", B, rng.randint(max(1, hi // 4), hi), hi, HKV, dtype=rng.choice(["bf16", "fp16"]))
    else:
        L = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
        hi = max(L, _log(rng, 50, 65536 if L <= 16 else min(16384, 10 ** 9 // (L * HQ))))
        B = max(1, min(_log(rng, 1, 32), 500000 // hi, 10 ** 9 // (L * hi * HQ)))
        c = _attend("", B, L, rng.randint(max(1, hi // 4), hi), hi, HQ, HKV, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    padded=L > 1 and rng.random() < 0.4)
    c.pop("name", None)
    return c


def _geometry(case):
    """Lengths of the sequences (with their new tokens), positions of the first new token, newest tokens of each.
    The same for every seed."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    B = case["B"]
    if case["kind"] == "append":
        pos = [case["before"]] + [r.randint(0, case["before"]) for _ in range(B - 1)]
        return {"lens": [p + case["T"] for p in pos], "pos": pos, "q": [case["T"]] * B}
    lens = [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(B - 1)]
    q = [min(case.get("L", 1), n) for n in lens]
    if case.get("padded"):
        q = [q[0]] + [r.randint(1, x) for x in q[1:]]
    return {"lens": lens, "pos": [n - x for n, x in zip(lens, q)], "q": q}


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _axes(case):
    """Frequency and axis of each of the 64 pairs."""
    sections = [int(x) for x in case["sections"].split(",")]
    if case["order"] == "blocks":
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    else:
        axis, left = [], list(sections)
        while len(axis) < D // 2:
            for a in range(len(sections)):
                if left[a]:
                    axis.append(a)
                    left[a] -= 1
    return len(sections), axis


def _positions(case, first):
    """Positions [axes, B, T]: frames of a video (time, height, width), rows of an image, or plain counts."""
    n, _ = _axes(case)
    B, T = case["B"], case["T"]
    side = max(1, int(math.sqrt(T / 4)))
    t = torch.arange(T, device="cuda").expand(B, T) + torch.as_tensor(first, device="cuda")[:, None]
    if n == 1:
        return t[None].contiguous()
    grid = torch.stack([t // (side * side), t // side % side, t % side])
    return (grid[3 - n:] + torch.as_tensor(first, device="cuda")[:, None]).contiguous()


def _tables(lens, seed):
    """Scattered pages of a pool for sequences of so many tokens."""
    pages = [-(-n // PAGE) for n in lens]
    perm = torch.randperm(sum(pages) + 1, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((len(lens), max(pages) + 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table.cuda(), sum(pages) + 1


def _pools(P, H, g):
    """Empty pools: whatever the memory held before (here random bytes)."""
    shapes = {"k": (P, H, PAGE, 64), "k_scale": (P, H, 4, PAGE), "v": (P, H, D, 32), "v_scale": (P, H, 4, PAGE)}
    return {name: torch.randint(0, 256, s, generator=g, device="cuda", dtype=torch.uint8) for name, s in shapes.items()}


def _held(x):
    """Values in 32 bits [..., 128] as the format holds them, and their scale bytes [..., 4]."""
    b = x.float().unflatten(-1, (4, BLOCK))
    top = b.abs().amax(-1)
    fraction, exponent = torch.frexp(top)  # top = fraction 2^exponent, fraction in [1/2, 1)
    e = (exponent - 3 + (fraction > 0.875)).clamp(_LOW - 127, _HIGH - 127)
    e = torch.where(top == 0, _LOW - 127, e)
    y = torch.ldexp(b, -e[..., None])
    a = y.abs().clamp_max(6)
    level = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), (a / 2).round() * 2))
    level = level.copysign(y)
    good = torch.isfinite(top)
    byte = torch.where(good, e + 127, _NAN).to(torch.uint8)
    return level, byte


def _codes(level):
    a = level.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    return c | (level.signbit().to(torch.uint8) << 3)


def _store(pools, pages, k, v):
    """Whole pages' tokens [n 64, H, 128] into the pools, in the pages' order."""
    n, H = pages.shape[0], k.shape[1]
    for name, x in (("k", k), ("v", v)):
        level, byte = _held(x)
        c = _codes(level).view(n, PAGE, H, D)
        if name == "k":  # [tile 4, block 4, row 16, byte 16]: token 4 row + tile
            c = c.view(n, 16, 4, H, 4, 16, 2)
            c = (c[..., 0] | c[..., 1] << 4).permute(0, 3, 2, 4, 1, 5).reshape(n, H, PAGE, 64)
        else:  # [pair of columns 4, tokens 4, column 16, 2, byte 8]: token 16 group + 2 byte + nibble
            c = c.view(n, 4, 8, 2, H, 4, 2, 16)
            c = (c[:, :, :, 0] | c[:, :, :, 1] << 4).permute(0, 3, 4, 1, 6, 5, 2).reshape(n, H, D, 32)
        pools[name][pages] = c
        pools[name + "_scale"][pages] = byte.view(n, PAGE, H, 4).permute(0, 2, 3, 1)


def _fill(pools, table, lens, g, heavy=None):
    """Random tokens into the sequences' pages; `heavy`(b, k, t0) may put keys there that queries look for."""
    H = pools["k"].shape[1]
    for b, n in enumerate(lens):
        pages = -(-n // PAGE)
        for c in range(0, pages, 512):  # in pieces of 32K tokens
            ids = table[b, c:min(c + 512, pages)].long()
            k = torch.randn((ids.shape[0] * PAGE, H, D), generator=g, device="cuda")
            v = torch.randn((ids.shape[0] * PAGE, H, D), generator=g, device="cuda")
            if heavy:
                heavy(b, k)
            _store(pools, ids, k, v)


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], _DT[case["dtype"]]
    B, HKV = case["B"], case["HKV"]
    st = {"case": case}
    if kind == "rotate":
        T = case["T"]
        st["q"] = torch.randn((B, T, case["HQ"], D), generator=g, device="cuda").to(dt)
        st["k"] = torch.randn((B, T, HKV, D), generator=g, device="cuda").to(dt)
        r = random.Random(seed)
        st["positions"] = _positions(case, [r.randint(0, case["far"]) for _ in range(B)])
    else:
        geo = st["geo"] = _geometry(case)
        st["T"] = max(geo["lens"])
        st["table"], P = _tables(geo["lens"], seed)
        st["lens"] = torch.tensor(geo["lens"], dtype=torch.int32, device="cuda")
        st["pools"] = _pools(P, HKV, g)
        heavy = None
        if kind == "attend":
            L, HQ = case["L"], case["HQ"]
            q = st["q"] = torch.randn((B, L, HQ, D), generator=g, device="cuda").to(dt)
            st["q_lens"] = torch.tensor(geo["q"], dtype=torch.int32, device="cuda") if min(geo["q"]) < L else None

            def heavy(b, k):  # keys that some of the queries look for (cosine 0.8), as trained attention has them
                n = min(16, k.shape[0])
                t = torch.randperm(k.shape[0], generator=g, device="cuda")[:n]
                i = torch.randint(0, L, (n,), generator=g, device="cuda")
                r = torch.randint(0, HQ // HKV, (n,), generator=g, device="cuda")
                look = q[b].view(L, HKV, HQ // HKV, D)[i, :, r].float()
                k[t] = 0.8 * math.sqrt(D) * look / look.norm(dim=-1, keepdim=True) + 0.6 * k[t]
        if kind == "append":
            T = case["T"]
            st["pos"] = torch.tensor(geo["pos"], dtype=torch.int32, device="cuda")
            if case["sections"]:
                st["q"] = torch.randn((B, T, case["HQ"], D), generator=g, device="cuda").to(dt)
                st["positions"] = _positions(case, geo["pos"])
            # keys with some channels far larger than the others, as trained projections have them
            gain = torch.exp(torch.randn((HKV, D), generator=g, device="cuda"))
            st["k"] = (torch.randn((B, T, HKV, D), generator=g, device="cuda") * gain).to(dt)
            st["v"] = torch.randn((B, T, HKV, D), generator=g, device="cuda").to(dt)
        _fill(st["pools"], st["table"], geo["lens"], g, heavy)
    if own:  # the handles that a program keeps
        p = str(Path(__file__).resolve().parents[1] / "ffa-speedtest_amd")
        if p not in sys.path:
            sys.path.insert(0, p)
        if case.get("sections"):
            from ffa_mi355x.rope_axes import AxisRope

            st["rope"] = AxisRope([int(x) for x in case["sections"].split(",")], device="cuda", pairs=case["pairs"],
                                  order=case["order"])
        if kind != "rotate":
            from ffa_mi355x.paged_mxfp4 import PagedMXFP4Cache

            cache = st["cache"] = PagedMXFP4Cache(P, HKV, "cuda")
            for name, t in st.pop("pools").items():
                getattr(cache, name).copy_(t)
    return st


# ---------------------------------------------------------------------------- the plain form
def _turn(case, positions, x):
    """x [B, T, H, 128] rotated (in 32 bits, its angles in 64)."""
    _, axis = _axes(case)
    f = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=x.device) / (D // 2))
    angle = positions[torch.tensor(axis, device=x.device)].permute(1, 2, 0).double() * f
    c, s = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    if case.get("inverse"):
        s = -s
    x = x.float()
    if case["pairs"] == "half":
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def _read(pools, table):
    """Keys and values [B, H, 64 columns, 128] of the table's pages, in 32 bits."""
    B, n = table.shape
    pages = table.reshape(-1).long()
    H = pools["k"].shape[1]
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=table.device)
    got = []
    for name in ("k", "v"):
        c = pools[name][pages]
        c = torch.stack([c & 15, c >> 4], -1)
        if name == "k":
            c = c.view(B, n, H, 4, 4, 16, 32).permute(0, 2, 1, 5, 3, 4, 6)
        else:
            c = c.view(B, n, H, 4, 4, 16, 2, 16).permute(0, 2, 1, 4, 7, 3, 6, 5)
        byte = pools[name + "_scale"][pages].view(B, n, H, 4, PAGE).permute(0, 2, 1, 4, 3).reshape(B, H, n * PAGE, 4, 1)
        scale = torch.ldexp(torch.ones((), device=c.device), byte.int() - 127).masked_fill(byte == _NAN, math.nan)
        got.append((levels[c.reshape(B, H, n * PAGE, 4, BLOCK).int()] * scale).flatten(-2))
    return got


def _plain_append(st):
    case, pools = st["case"], st["pools"]
    k, v = st["k"].float(), st["v"].float()
    if case["sections"]:
        k = _turn(case, st["positions"], k)
    B, T, H, _ = k.shape
    pos = st["pos"][:, None].long() + torch.arange(T, device=k.device)
    page, t = st["table"].long().gather(1, pos // PAGE)[..., None, None], (pos % PAGE)[..., None, None]
    head = torch.arange(H, device=k.device)[:, None]
    out = []
    for name, x in (("k", k), ("v", v)):
        level, byte = _held(x)
        c = _codes(level).flatten(-2)
        if name == "k":  # two channels of a token to a byte
            b = torch.arange(64, device=k.device)
            at = (t % 4 * 64 + b // 16 * 16 + t // 4) * 16 + b % 16
            pools["k"].view(-1, H, 4096)[page, head, at] = c[..., ::2] | c[..., 1::2] << 4
        else:  # two tokens of a channel: each into its half of the byte, even ones first
            ch = torch.arange(D, device=k.device)
            at = (ch // 32 * 64 + t // 16 * 16 + ch % 16) * 16 + ch // 16 % 2 * 8 + t % 16 // 2
            flat = pools["v"].view(-1)
            where = (page * H + head) * 4096 + at
            odd = (t % 2 == 1).expand_as(where)
            flat[where[~odd]] = flat[where[~odd]] & 240 | c[~odd]
            flat[where[odd]] = flat[where[odd]] & 15 | c[odd] << 4
        pools[name + "_scale"][page, head, torch.arange(4, device=k.device), t] = byte
        scale = torch.ldexp(torch.ones((), device=k.device), byte.int() - 127).masked_fill(byte == _NAN, math.nan)
        out.append((level * scale[..., None]).flatten(-2).to(st["k"].dtype))
    return out


def _plain_readback(st):
    dt = _DT[st["case"]["dtype"]]
    n = -(-st["T"] // PAGE)
    past = torch.arange(n * PAGE, device="cuda")[None, None, :, None] >= st["lens"][:, None, None, None]
    return [x.masked_fill(past, 0).transpose(1, 2).to(dt).contiguous() for x in _read(st["pools"], st["table"][:, :n])]


def _plain_attend(st):
    q, lens = st["q"], st["lens"]
    B, L, HQ, _ = q.shape
    H = st["case"]["HKV"]
    k, v = _read(st["pools"], st["table"][:, :-(-st["T"] // PAGE)])
    q_lens = torch.full_like(lens, L) if st["q_lens"] is None else st["q_lens"]
    t = torch.arange(k.shape[2], device=q.device)
    v = v.masked_fill((t >= lens[:, None])[:, None, :, None], 0)  # slots that hold no token yet
    i = torch.arange(L, device=q.device)
    sees = (lens - q_lens)[:, None] + i + 1  # keys below this
    sees = torch.where(i < q_lens[:, None], sees, 0).repeat_interleave(HQ // H, 1)[:, None, :, None]
    x = q.float().view(B, L, H, -1, D).transpose(1, 2).reshape(B, H, -1, D)
    s = (x @ k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D)).masked_fill_(t >= sees, -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(B, H, L, -1, D).transpose(1, 2).reshape(B, L, HQ, D).to(q.dtype)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        if kind == "rotate":
            return st["rope"].rotate(st["positions"], st["q"], st["k"], inverse=case["inverse"])
        cache = st["cache"]
        if kind == "readback":
            return cache.dequantize(st["table"], st["T"], st["lens"], out_dtype=_DT[case["dtype"]])
        if kind == "attend":
            return cache.attend(st["q"], st["table"], st["lens"], T=st["T"], q_lens=st["q_lens"])
        if case["sections"]:
            return cache.append_rotary(st["q"], st["k"], st["v"], st["pos"], st["table"], st["rope"], st["positions"],
                                       values=True, check=False)
        cache.append(st["k"], st["v"], st["pos"], st["table"], check=False)
        return cache.dequantize(st["table"], st["T"], st["lens"], out_dtype=_DT[case["dtype"]])
    if kind == "rotate":
        return [_turn(case, st["positions"], x).to(x.dtype) for x in (st["q"], st["k"])]
    if kind == "readback":
        return _plain_readback(st)
    if kind == "attend":
        return _plain_attend(st)
    if case["sections"]:
        return [_turn(case, st["positions"], st["q"]).to(st["q"].dtype)] + _plain_append(st)
    _plain_append(st)
    return _plain_readback(st)


# ---------------------------------------------------------------------------- work, and the definition in 64 bits
def work(case):
    kind, HKV, es = case["kind"], case["HKV"], 4 if case["dtype"] == "fp32" else 2
    token = 2 * (64 + 4)  # codes and scales of a token and head
    if kind == "rotate":
        n = case["B"] * case["T"]
        return {"bytes": n * (case["HQ"] + HKV) * D * es * 2 + 8 * n * _axes(case)[0], "flops": 3 * n * (case["HQ"] + HKV) * D}
    geo = _geometry(case)
    if kind == "append":
        n = case["B"] * case["T"]
        new = n * HKV * (2 * D * es + token)
        if case["sections"]:
            return {"bytes": new + n * 2 * D * es * (case["HQ"] + HKV), "flops": 3 * n * (case["HQ"] + HKV) * D}
        padded = case["B"] * -(-max(geo["lens"]) // PAGE) * PAGE
        return {"bytes": new + (sum(geo["lens"]) - n) * HKV * token + padded * HKV * 2 * D * es, "flops": 0}
    if kind == "readback":
        padded = case["B"] * -(-max(geo["lens"]) // PAGE) * PAGE
        return {"bytes": sum(geo["lens"]) * HKV * token + padded * HKV * 2 * D * es, "flops": 0}
    flops = sum(4 * D * case["HQ"] * (q * n - q * (q - 1) // 2) for n, q in zip(geo["lens"], geo["q"]))
    return {"bytes": sum(geo["lens"]) * HKV * token + 2 * sum(geo["q"]) * case["HQ"] * D * es, "flops": flops}


def _rotated64(case, positions, x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    _, axis = _axes(case)
    for j, a in enumerate(axis):
        angle = positions[a].double() * 10000.0 ** (-j / 64)
        angle = -angle if case.get("inverse") else angle
        c, s = torch.cos(angle)[..., None], torch.sin(angle)[..., None]
        m, n = (j, j + 64) if case["pairs"] == "half" else (2 * j, 2 * j + 1)
        u, w = x[..., m].double(), x[..., n].double()
        out[..., m] = u * c - w * s
        out[..., n] = w * c + u * s
    return out


def _held64(x):
    """The format's value nearest to each of x (64 bits), by its definition."""
    b = x.double().reshape(-1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.full_like(top, -22.0)
    for k in range(-21, 14):  # the smallest power of two of which the largest value is at most seven
        e = torch.where(top > 7 * 2.0 ** (k - 1), float(k), e)
    y = b / 2.0 ** e
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    got = torch.zeros_like(y)
    for i in range(7):  # past a midpoint, or on it where the level above has an even code
        mid = (levels[i] + levels[i + 1]) / 2
        got = torch.where(y.abs() >= mid if i % 2 else y.abs() > mid, levels[i + 1], got)
    return (got * y.sign() * 2.0 ** e).reshape(x.shape)


def _elements(pools, pages, head):
    """Keys and values [64 n, 128] of one head, element by element of the pages' stated order, in 64 bits."""
    dev = pages.device
    t, c = torch.arange(PAGE, device=dev)[:, None], torch.arange(D, device=dev)[None, :]
    at_k, half_k = ((t & 3) * 64 + (c >> 5) * 16 + (t >> 2)) * 16 + (c >> 1 & 15), (c & 1).expand(PAGE, D)
    at_v, half_v = ((c >> 5) * 64 + (t >> 4) * 16 + (c & 15)) * 16 + (c >> 4 & 1) * 8 + (t >> 1 & 7), (t & 1).expand(PAGE, D)
    at_s = ((c >> 5) * PAGE + t).reshape(-1)
    got = []
    for name, at, half in (("k", at_k, half_k), ("v", at_v, half_v)):
        code = pools[name][pages, head].reshape(len(pages), -1)[:, at.reshape(-1)].int() >> (4 * half.reshape(-1)) & 15
        byte = pools[name + "_scale"][pages, head].reshape(len(pages), -1)[:, at_s].double()
        m, x = (code & 1).double(), (code >> 1 & 3).double()
        value = torch.where(x == 0, m / 2, (1 + m / 2) * 2.0 ** (x - 1)) * 2.0 ** (byte - 127)
        got.append(torch.where(code > 7, -value, value).reshape(-1, D))
    return got


def exact(case, seed):
    """The definition in 64 bits."""
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    kind = case["kind"]
    if kind == "rotate":
        return [_rotated64(case, st["positions"], st[x]) for x in ("q", "k")]
    if kind == "append" and case["sections"]:
        return [_rotated64(case, st["positions"], st["q"]), _held64(_rotated64(case, st["positions"], st["k"])), _held64(st["v"])]
    H, table, lens = case["HKV"], st["table"], st["geo"]["lens"]
    if kind != "attend":
        T = -(-st["T"] // PAGE) * PAGE
        out = [torch.zeros((case["B"], T, H, D), dtype=torch.float64, device="cuda") for _ in range(2)]
        for b, n in enumerate(lens):
            for h in range(H):
                for o, x in zip(out, _elements(st["pools"], table[b, :-(-n // PAGE)].long(), h)):
                    o[b, :n, h] = x[:n]
            if kind == "append":
                p = st["geo"]["pos"][b]
                out[0][b, p:n], out[1][b, p:n] = _held64(st["k"][b]), _held64(st["v"][b])
        return out
    q = st["q"]
    G = case["HQ"] // H
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, (n, ql) in enumerate(zip(lens, st["geo"]["q"])):
        for h in range(H):
            k, v = (x[:n] for x in _elements(st["pools"], table[b, :-(-n // PAGE)].long(), h))
            for r in range(G):
                for a in range(0, ql, 512):
                    e = min(a + 512, ql)
                    s = q[b, a:e, h * G + r].double() @ k.T / math.sqrt(D)
                    row = torch.arange(n - ql + a, n - ql + e, device="cuda")[:, None]
                    s = s.masked_fill(torch.arange(n, device="cuda")[None, :] > row, -math.inf)
                    out[b, a:e, h * G + r] = torch.softmax(s, dim=-1) @ v
    return out
