"""The operators for several sequences out of one prompt, as measured cases.

Three kinds of call on the paged quantized caches (64-token pages):

  attend  exact attention of the L newest tokens of every sequence over its cached keys and values: decode
          steps that must not prune, drafted tokens, a prompt's next chunk
  shared  the same for groups of sequences that share the leading pages of their block tables (a system
          prompt, samples or beams of one request): those pages count once per group
  pages   management of the pages of several layers' caches: copying, forking sequences (and freeing them
          again), compacting the pool

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
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_NF4 = (-1.0, -0.6961928009986877, -0.5229921340942383, -0.39491748809814453, -0.28444138169288635,
        -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
        0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)


# ---------------------------------------------------------------------------- the cases
def _attend(name, fmt, B, L, lo, hi, HQ=32, HKV=8, dtype="bf16", res="e4m3", v="fp16", padded=False):
    return {"name": name, "kind": "attend", "fmt": fmt, "B": B, "L": L, "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV,
            "dtype": dtype, "res": res, "v": v, "padded": padded}


def _shared(name, fmt, groups, members, even, prefix, own_hi, L=1, HQ=32, HKV=8, dtype="bf16", res="e4m3", v="fp16"):
    return {"name": name, "kind": "shared", "fmt": fmt, "groups": groups, "members": members, "even": even,
            "prefix": prefix, "own_hi": own_hi, "L": L, "HQ": HQ, "HKV": HKV, "dtype": dtype, "res": res, "v": v}


def listed():
    return [
        # one short conversation, one token: latency
        _attend("attend_b1_2k", "q2", 1, 1, 2000, 2000),
        # a serving batch of long, ragged contexts, one token each: the caches' bytes
        _attend("attend_b16_ragged", "q2", 16, 1, 8192, 65536),
        # five drafted tokens of each of eight sequences on the 4-bit cache
        _attend("attend_draft_nf4_b8", "nf4", 8, 5, 8192, 65536),
        # the last 2K tokens of a 16K prompt: a chunk of a long prefill
        _attend("attend_chunk_2k_of_16k", "q2", 1, 2048, 16384, 16384),
        # three prompts of different lengths in one padded batch, 64 query heads
        _attend("attend_prompts_b3", "nvfp4", 3, 701, 300, 701, HQ=64, dtype="fp16", res="e5m2", padded=True),
        # four beams of one short request: latency
        _shared("shared_beams", "q2", 1, 4, True, 2000, 40),
        # a serving batch behind one 32K-token document, each with an answer of up to 2K tokens of its own
        _shared("shared_b64_32k", "q2", 1, 64, True, 32768, 2000),
        # five requests with up to 24 samples each, 64 query heads, the nvfp4 cache
        _shared("shared_groups_nvfp4", "nvfp4", 5, 24, False, 9000, 600, HQ=64, dtype="fp16"),
        # five drafted tokens of 16 sequences behind 64K tokens, residual e5m2, bf16 values
        _shared("shared_draft_64k", "q2", 1, 16, True, 65536, 500, L=5, res="e5m2", v="bf16"),
        # three pages of one layer: latency
        {"name": "pages_copy_3", "kind": "pages", "op": "copy", "fmt": "q2", "layers": 1, "HKV": 8, "P": 64, "n": 3,
         "hi": 0},
        # 64 children of 8 sequences of some 4K tokens, in 8 layers, freed again
        {"name": "pages_fork_b64", "kind": "pages", "op": "fork", "fmt": "q2", "layers": 8, "HKV": 8, "P": 640, "n": 64,
         "hi": 4096},
        # a pool of 4 layers, half of its pages free, packed into its lower half
        {"name": "pages_compact_1k", "kind": "pages", "op": "compact", "fmt": "nvfp4", "layers": 4, "HKV": 8, "P": 1024,
         "n": 16, "hi": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "shared", "shared", "shared", "pages"])
    fmt = rng.choice(["q2", "q2", "nvfp4", "nf4"])
    types = {"dtype": rng.choice(["bf16", "bf16", "fp16"]), "res": rng.choice(["e4m3", "e4m3", "e5m2"]),
             "v": rng.choice(["fp16", "fp16", "bf16"])}
    HKV = rng.choice([1, 2, 4, 8, 8])
    HQ = HKV * rng.choice([1, 2, 4, 4, 7, 8])
    if kind == "attend":
        L = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
        hi = max(L, _log(rng, 50, 65536 if L <= 16 else min(16384, 10 ** 9 // (L * HQ))))
        B = max(1, min(_log(rng, 1, 32), 500000 // hi, 10 ** 9 // (L * hi * HQ)))
        lo = rng.randint(max(1, hi // 4), hi)
        c = _attend("", fmt, B, L, lo, hi, HQ, HKV, padded=L > 1 and rng.random() < 0.4, **types)
    elif kind == "shared":
        L = rng.choice([1, 1, 1, _log(rng, 2, 8)])
        groups = rng.choice([1, 1, 2, 5])
        prefix = _log(rng, 64, 32768 // groups)
        members = _log(rng, 2, max(2, min(64, 4096 * 64 // (prefix * L) + 8)))
        c = _shared("", fmt, groups, members, rng.random() < 0.5, prefix, _log(rng, 1, 2000), L, HQ, HKV, **types)
    else:
        op = rng.choice(["copy", "fork", "compact"])
        layers = rng.choice([1, 2, 8])
        P = _log(rng, 64, 4096 // layers)
        c = {"kind": "pages", "op": op, "fmt": fmt, "layers": layers, "HKV": HKV, "P": P,
             "n": _log(rng, 1, P // 4), "hi": _log(rng, 1, 16 * P)}
    c.pop("name", None)
    return c


def _lens(case):
    """Lengths of the sequences, whole; of their own tokens past the shared ones; the groups' sizes and shared
    tokens; the newest tokens of each.  The same for every seed."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "attend":
        lens = [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["B"] - 1)]
        q = [min(case["L"], n) for n in lens]
        if case["padded"]:
            q = [q[0]] + [r.randint(1, x) for x in q[1:]]
        return {"lens": lens, "sizes": [1] * case["B"], "prefix": [0] * case["B"], "q": q}
    sizes, prefix, lens = [], [], []
    for g in range(case["groups"]):
        sizes.append(case["members"] if case["even"] or g == 0 else r.randint(1, case["members"]))
        prefix.append(case["prefix"] if case["even"] or g == 0 else r.randint(max(1, case["prefix"] // 8), case["prefix"]))
        lens += [prefix[-1] + r.randint(max(1, case["own_hi"] // 32), case["own_hi"]) for _ in range(sizes[-1])]
    lens = [max(n, case["L"]) for n in lens]
    return {"lens": lens, "sizes": sizes, "prefix": prefix, "q": [case["L"]] * len(lens)}


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pools(fmt, P, HKV, res, v, g):
    """Empty pools: whatever the memory held before (here random bytes)."""
    shapes = {"q2": [("k_q", (P, HKV, 4, PAGE, 8), torch.uint8), ("k_scale", (P, HKV, 4, PAGE), torch.float16),
                     ("k_zero", (P, HKV, 4, PAGE), torch.float16)],
              "nvfp4": [("k", (P, HKV, PAGE, 64), torch.uint8), ("k_scale", (P, HKV, PAGE, 8), torch.float8_e4m3fn)],
              "nf4": [("k", (P, HKV, PAGE, 64), torch.uint8), ("k_scale", (P, HKV, PAGE, 2), torch.float16)]}[fmt]
    shapes = shapes + [("k_res", (P, HKV, PAGE, D), _FP8[res]), ("v", (P, HKV, D, PAGE), _DT[v])]
    out = {}
    for name, shape, dt in shapes:
        n = math.prod(shape) * torch.empty((), dtype=dt).element_size()
        words = torch.randint(-2 ** 63, 2 ** 63 - 1, ((n + 7) // 8,), generator=g, device="cuda")
        out[name] = words.view(torch.uint8)[:n].view(dt).view(shape)
    return out


def _fill(fmt, pools, pages, k, v):
    """Quantize k [T, HKV, D] (T a multiple of 64) and store it with v in the pages."""
    n, H = pages.shape[0], k.shape[1]
    f8 = pools["k_res"].dtype
    if fmt == "q2":
        x = k.view(-1, H, 4, 32)
        zero = x.amin(-1).half()
        scale = ((x.amax(-1) - zero.float()).clamp_min(1e-6) / 3).half()
        c = torch.round((x - zero.float()[..., None]) / scale.float()[..., None]).clamp_(0, 3)
        base = (c * scale.float()[..., None] + zero.float()[..., None]).view(-1, H, D)
        c = c.to(torch.uint8).view(n, 16, 2, 2, H, 4, 8, 4)  # page, m, h, t & 1, head, group, byte, code
        b = c[..., 0] | c[..., 1] << 2 | c[..., 2] << 4 | c[..., 3] << 6
        pools["k_q"][pages] = b.permute(0, 4, 2, 5, 1, 3, 6).reshape(n, H, 4, PAGE, 8)
        for name, t in (("k_scale", scale), ("k_zero", zero)):  # token 16 kc + 4 m + 2 h + l
            pools[name][pages] = t.view(n, 4, 4, 2, 2, H, 4).permute(0, 5, 3, 6, 1, 4, 2).reshape(n, H, 4, PAGE)
    else:
        w = 16 if fmt == "nvfp4" else 64
        x = k.view(-1, H, D // w, w)
        amax = x.abs().amax(-1)
        if fmt == "nvfp4":
            scale = (amax / 6).clamp(2 ** -9, 448).to(torch.float8_e4m3fn)
            levels = torch.tensor(_E2M1[:0:-1], device=k.device).neg().tolist() + list(_E2M1)
            code_of = torch.tensor(list(range(15, 8, -1)) + list(range(8)), dtype=torch.uint8, device=k.device)
        else:
            scale = amax.clamp_min(1e-6).half()
            levels, code_of = list(_NF4), torch.arange(16, dtype=torch.uint8, device=k.device)
        lv = torch.tensor(levels, device=k.device)
        i = torch.bucketize(x / scale.float()[..., None], (lv[1:] + lv[:-1]) / 2)
        base = (lv[i] * scale.float()[..., None]).view(-1, H, D)
        c = code_of[i].view(n, 16, 4, H, 4, 16, 2)  # page, m, tau, head, kc, byte, nibble
        pools["k"][pages] = (c[..., 0] | c[..., 1] << 4).permute(0, 3, 2, 4, 1, 5).reshape(n, H, PAGE, 64)
        s = scale.view(n, PAGE, H, D // w).transpose(1, 2)
        if fmt == "nvfp4":
            pools["k_scale"].view(torch.uint8)[pages] = s.contiguous().view(torch.uint8)
        else:
            pools["k_scale"][pages] = s
    r = (k - base).to(f8).view(torch.uint8).view(n, 16, 4, H, 4, 2, 16)  # page, m, tau, head, kc, h, channel
    pools["k_res"].view(torch.uint8)[pages] = r.permute(0, 3, 2, 5, 4, 1, 6).reshape(n, H, PAGE, D)
    vt = v.to(pools["v"].dtype).view(n, 4, 2, 8, H, 8, 16)  # page, kc, kap, token, head, nu, column
    pools["v"][pages] = vt.permute(0, 4, 5, 2, 1, 6, 3).reshape(n, H, D, PAGE)


def _attention_inputs(case, seed):
    g = _gen(seed)
    geo = _lens(case)
    HQ, HKV, L = case["HQ"], case["HKV"], case["L"]
    G, B, dt = HQ // HKV, len(geo["lens"]), _DT[case["dtype"]]
    q = torch.randn((B, L, HQ, D), generator=g, device="cuda").to(dt)
    # every sequence's pages: the group's shared whole pages, then its own (the last partial page of the common
    # prompt is its own copy, as forking leaves it)
    np_ = [-(-n // PAGE) for n in geo["lens"]]
    shared = [p // PAGE for p in geo["prefix"]]
    runs, b = [], 0  # (first sequence, sequences, first page, pages)
    for n, sp in zip(geo["sizes"], shared):
        if sp:
            runs.append((b, n, 0, sp))
        runs += [(i, 1, sp, np_[i] - sp) for i in range(b, b + n) if np_[i] > sp]
        b += n
    total = sum(r[3] for r in runs)
    perm = torch.randperm(total + 1, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((B, max(np_) + 1), dtype=torch.int32)
    pools = _pools(case["fmt"], total + 1, HKV, case["res"], case["v"], g)
    at = 0
    for b0, n, p0, pg in runs:
        ids = perm[at:at + pg]
        at += pg
        table[b0:b0 + n, p0:p0 + pg] = ids
        for c in range(0, pg, 512):  # in pieces of 32K tokens
            m = min(512, pg - c)
            k = torch.randn((m * PAGE, HKV, D), generator=g, device="cuda")
            v = torch.randn((m * PAGE, HKV, D), generator=g, device="cuda")
            # keys that some of the queries look for (cosine 0.8), as trained attention has them
            heavy = min(16, m * PAGE)
            t = torch.randperm(m * PAGE, generator=g, device="cuda")[:heavy]
            qb = torch.randint(b0, b0 + n, (heavy,), generator=g, device="cuda")
            ql = torch.randint(0, L, (heavy,), generator=g, device="cuda")
            qr = torch.randint(0, G, (heavy,), generator=g, device="cuda")
            look = q.view(B, L, HKV, G, D)[qb, ql, :, qr].float()
            look = look / look.norm(dim=-1, keepdim=True)
            k[t] = 0.8 * math.sqrt(D) * look + 0.6 * k[t]
            _fill(case["fmt"], pools, ids[c:c + m].long().cuda(), k, v)
    st = {"case": case, "geo": geo, "q": q, "pools": pools, "table": table.cuda(), "T": max(geo["lens"]),
          "lens": torch.tensor(geo["lens"], dtype=torch.int32, device="cuda"), "shared": shared,
          "q_lens": torch.tensor(geo["q"], dtype=torch.int32, device="cuda") if min(geo["q"]) < L else None}
    return st


def _page_inputs(case, seed):
    g = _gen(seed)
    r = random.Random(seed)
    P, n, op = case["P"], case["n"], case["op"]
    pools = [_pools(case["fmt"], P, case["HKV"], "e4m3", "fp16", g) for _ in range(case["layers"])]
    refs = [0] * P
    st = {"case": case, "pools": pools}
    order = r.sample(range(P), P)
    if op == "copy":
        n = min(n, P // 2)
        st["src"] = torch.tensor(order[:n], dtype=torch.int32, device="cuda")
        st["dst"] = torch.tensor(order[n:2 * n], dtype=torch.int32, device="cuda")
        refs = [1] * P
    elif op == "fork":
        # some sequences fill up to half of the pool; n children of them
        hi = min(case["hi"], P * PAGE // 4)
        lens, used = [], 0
        while len(lens) < max(1, n // 8) and used + -(-hi // PAGE) <= P // 2:
            lens.append(r.randint(max(1, hi // 2), hi))
            used += -(-lens[-1] // PAGE)
        table = torch.full((len(lens), -(-hi // PAGE) + 2), -1, dtype=torch.int32)
        at = 0
        for b, x in enumerate(lens):
            k = -(-x // PAGE)
            table[b, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
            at += k
        for p in order[:at]:
            refs[p] = 1
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["parents"] = torch.tensor([r.randrange(len(lens)) for _ in range(n)], dtype=torch.int32, device="cuda")
        st["table"] = table.cuda()
    else:
        # n sequences over half of the pool; some of their pages are held twice
        live = order[:P // 2]
        cols = -(-len(live) // n)
        table = torch.full((n, cols + 1), -1, dtype=torch.int32)
        for i, p in enumerate(live):
            refs[p] = 1
            table[i // cols, i % cols] = p
        for b in range(1, n, 2):
            if int(table[b, 0]) >= 0:
                refs[int(table[b, 0])] -= 1
                table[b, 0] = table[b - 1, 0]
                refs[int(table[b - 1, 0])] += 1
        st["table"] = table.cuda()
    st["refs"] = torch.tensor(refs, dtype=torch.int32, device="cuda")
    return st


def _cache(fmt, pools):
    """The framework's cache over the pools."""
    from ffa_mi355x.paged import PagedQ2Cache
    from ffa_mi355x.paged_kfmt import PagedKfmtCache

    P, HKV = pools["v"].shape[:2]
    kw = {"res_dtype": pools["k_res"].dtype, "v_dtype": pools["v"].dtype}
    cache = PagedQ2Cache(P, HKV, "cuda", **kw) if fmt == "q2" else PagedKfmtCache(fmt, P, HKV, "cuda", **kw)
    for name, t in pools.items():
        getattr(cache, name).view(torch.uint8).copy_(t.view(torch.uint8))
    return cache


def prepare(case, seed):
    st = _page_inputs(case, seed) if case["kind"] == "pages" else _attention_inputs(case, seed)
    if own:
        p = str(Path(__file__).resolve().parents[1] / "ffa-speedtest_amd")
        if p not in sys.path:
            sys.path.insert(0, p)
        if case["kind"] == "pages":
            from ffa_mi355x.pages import PagePool

            caches = [_cache(case["fmt"], p) for p in st.pop("pools")]
            st["pool"] = PagePool(caches)
            st["pool"].refs.copy_(st["refs"])
            st["bytes"] = [t.view(torch.uint8) for c in caches for t in c.pools()]
        else:
            st["cache"] = _cache(case["fmt"], st.pop("pools"))
            if case["kind"] == "shared":
                from ffa_mi355x.attend import SharedPrefix

                st["plan"] = SharedPrefix(st["table"], st["lens"], group_sizes=st["geo"]["sizes"])
    elif case["kind"] == "pages":
        st["now"] = st["refs"].clone()
        st["bytes"] = [t.view(torch.uint8) for p in st["pools"] for t in p.values()]
    return st


# ---------------------------------------------------------------------------- the plain form
def _dequant(fmt, pools, pages):
    """K and V [HKV, 64 pages, D] of the pages, in 32 bits."""
    n, H = pages.shape[0], pools["v"].shape[1]
    if fmt == "q2":
        b = pools["k_q"][pages].view(n, H, 2, 4, 16, 2, 8, 1)  # h, group, m, t & 1, byte
        c = (b >> torch.tensor([0, 2, 4, 6], dtype=torch.uint8, device=b.device)) & 3
        c = c.permute(1, 0, 4, 2, 5, 3, 6, 7).reshape(H, n * PAGE, 4, 32).float()
        s, z = (pools[x][pages].view(n, H, 2, 4, 4, 2, 4).permute(1, 0, 4, 6, 2, 5, 3).reshape(H, n * PAGE, 4, 1).float()
                for x in ("k_scale", "k_zero"))
        k = c * s + z
    else:
        b = pools["k"][pages].view(n, H, 4, 4, 16, 16, 1)  # tau, kc, m, byte
        c = (b >> torch.tensor([0, 4], dtype=torch.uint8, device=b.device)) & 15
        c = c.permute(1, 0, 4, 2, 3, 5, 6).reshape(H, n * PAGE, D)
        lv = torch.tensor(_NF4 if fmt == "nf4" else _E2M1 + tuple(-x for x in _E2M1), device=b.device)
        s = pools["k_scale"].view(torch.uint8)[pages].view(pools["k_scale"].dtype).float()
        s = s.transpose(0, 1).reshape(H, n * PAGE, -1, 1)
        k = lv[c.int()].view(H, n * PAGE, s.shape[2], -1) * s
    r = pools["k_res"].view(torch.uint8)[pages].view(pools["k_res"].dtype).float().view(n, H, 4, 2, 4, 16, 16)
    k = k.reshape(H, n * PAGE, D) + r.permute(1, 0, 5, 2, 4, 3, 6).reshape(H, n * PAGE, D)
    v = pools["v"][pages].float().view(n, H, 8, 2, 4, 16, 8)  # nu, kap, kc, column, token
    return k, v.permute(1, 0, 4, 3, 6, 2, 5).reshape(H, n * PAGE, D)


def _plain_attention(st):
    case, geo, q = st["case"], st["geo"], st["q"]
    B, L, HQ, _ = q.shape
    H = case["HKV"]
    out = torch.zeros_like(q)
    b = 0
    for n, sp in zip(geo["sizes"], st["shared"]):
        if sp:
            kp, vp = _dequant(case["fmt"], st["pools"], st["table"][b, :sp].long())
        for i in range(b, b + n):
            T, ql = geo["lens"][i], geo["q"][i]
            parts = []
            if T > sp * PAGE:
                ko, vo = _dequant(case["fmt"], st["pools"], st["table"][i, sp:-(-T // PAGE)].long())
                parts = [(sp * PAGE, ko[:, :T - sp * PAGE], vo[:, :T - sp * PAGE])]
            if sp:
                parts.append((0, kp, vp))
            x = q[i, :ql].float().view(ql, H, -1, D).transpose(0, 1).reshape(H, -1, D)  # [H, ql * G, D]
            pos = torch.arange(T - ql, T, device=q.device).repeat_interleave(HQ // H)
            s = [(x @ k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(D)).masked_fill_(
                torch.arange(t0, t0 + k.shape[1], device=q.device) > pos[:, None], -math.inf) for t0, k, _ in parts]
            top = torch.stack([y.amax(-1, keepdim=True) for y in s]).amax(0)
            p = [(y - top).exp_() for y in s]
            o = sum(y @ v for y, (_, _, v) in zip(p, parts)) / sum(y.sum(-1, keepdim=True) for y in p)
            out[i, :ql] = o.view(H, ql, -1, D).transpose(0, 1).reshape(ql, HQ, D).to(q.dtype)
        b += n
    return out


def _plain_fork(st):
    refs, table, lens, parents = st["now"], st["table"], st["lens"], st["parents"].long()
    child, n = table[parents], lens[parents].long()
    col = torch.arange(table.shape[1], device=table.device)
    child = torch.where(col < -(-n // PAGE)[:, None], child, -1)
    rows = torch.nonzero(n % PAGE).view(-1)
    src = child[rows, n[rows] // PAGE].long()
    dst = torch.nonzero(refs == 0).view(-1)[:rows.shape[0]]
    held = child[col < (n // PAGE)[:, None]].long()
    refs += torch.bincount(held, minlength=refs.shape[0]).int()
    refs[dst] = 1
    child[rows, n[rows] // PAGE] = dst.int()
    for pools in st["pools"]:
        for t in pools.values():
            t = t.view(torch.uint8)
            t[dst] = t[src]
    held = child[col < -(-n // PAGE)[:, None]].long()  # the children's pages, freed again
    after = refs.clone()
    refs -= torch.bincount(held, minlength=refs.shape[0]).int()
    return child, after, refs


def _plain_compact(st):
    refs, table = st["now"], st["table"].clone()
    live = refs > 0
    low = torch.arange(refs.shape[0], device=refs.device) < live.sum()
    dst, src = torch.nonzero(low & ~live).view(-1), torch.nonzero(live & ~low).view(-1)
    to = torch.arange(refs.shape[0], dtype=torch.int32, device=refs.device)
    to[src] = dst.int()
    table = torch.where(table >= 0, to[table.clamp_min(0).long()], table)
    refs[dst] = refs[src]
    refs[src] = 0
    for pools in st["pools"]:
        for t in pools.values():
            t = t.view(torch.uint8)
            t[dst] = t[src]
    return table, refs


def run(st):
    case = st["case"]
    if case["kind"] in ("attend", "shared"):
        if own:
            return st["cache"].attend(st["q"], st["table"], st["lens"], T=st["T"], q_lens=st["q_lens"],
                                      shared=st.get("plan"))
        return _plain_attention(st)
    if case["op"] == "copy":
        if own:
            st["pool"].copy(st["src"], st["dst"], check=False)
        else:
            src, dst = st["src"].long(), st["dst"].long()
            for t in st["bytes"]:
                t[dst] = t[src]
        return st["bytes"]
    if case["op"] == "fork":
        if own:
            pool = st["pool"]
            child = pool.fork(st["table"], st["lens"], st["parents"], check=False)
            after = pool.refs.clone()
            pool.free(child, st["lens"][st["parents"]], check=False)
            return [child, after, pool.refs] + st["bytes"]
        return list(_plain_fork(st)) + st["bytes"]
    # each pass packs the same pool: its counts are set back first
    if own:
        pool = st["pool"]
        pool.refs.copy_(st["refs"])
        table = st["table"].clone()
        pool.compact(table, check=False)
        return [table, pool.refs] + st["bytes"]
    st["now"].copy_(st["refs"])
    return list(_plain_compact(st)) + st["bytes"]


# ---------------------------------------------------------------------------- work, and the definition in 64 bits
def work(case):
    HKV = case["HKV"]
    token = {"q2": 48, "nvfp4": 72, "nf4": 68}[case["fmt"]] + D + 2 * D  # K codes and scales, residual, V
    if case["kind"] == "pages":
        page = PAGE * HKV * token * case["layers"]
        if case["op"] == "copy":
            n = min(case["n"], case["P"] // 2)
        elif case["op"] == "fork":
            n = case["n"]
        else:
            n = case["P"] // 4
        return {"bytes": 2 * n * page + 4 * case["P"], "flops": 0}
    geo = _lens(case)
    tokens, flops, b = 0, 0, 0
    for n, p in zip(geo["sizes"], geo["prefix"]):
        sp = p // PAGE * PAGE
        tokens += sp
        for i in range(b, b + n):
            T, q = geo["lens"][i], geo["q"][i]
            tokens += T - sp
            flops += 4 * D * case["HQ"] * (q * T - q * (q - 1) // 2)
        b += n
    return {"bytes": tokens * HKV * token + 2 * sum(geo["q"]) * case["HQ"] * D * 2, "flops": flops}


def exact(case, seed):
    """The definition, token by token of the pages' stated layout, in 64 bits."""
    if case["kind"] == "pages":
        return None
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    fmt, pools, geo, q = case["fmt"], st["pools"], st["geo"], st["q"]
    dev, H = q.device, case["HKV"]
    G = case["HQ"] // H
    t = torch.arange(PAGE, device=dev)[:, None]
    c = torch.arange(D, device=dev)[None, :]
    # where element (token t, channel c) of a (page, head) block lies
    at_res = (((t & 3) * 2 + ((c >> 4) & 1)) * 64 + (c >> 5) * 16 + (t >> 2)) * 16 + (c & 15)
    at_v = (((c >> 4) * 2 + ((t >> 3) & 1)) * 64 + (t >> 4) * 16 + (c & 15)) * 8 + (t & 7)
    slot = 16 * (t // 16) + 4 * (t % 4) + (t // 4) % 4
    at_s = ((((slot >> 3) & 1) * 4 + (c >> 5)) * 4 + (slot >> 4)) * 8 + (slot & 7)
    at_2 = (((((t >> 1) & 1) * 64 + (c >> 5) * 16 + (t >> 2)) * 2 + (t & 1)) * 8) + ((c & 31) >> 2)
    at_4 = ((t & 3) * 64 + (c >> 5) * 16 + (t >> 2)) * 16 + ((c & 31) >> 1)

    def element(pool, pages, head, at):
        block = pool.view(pool.shape[0], H, -1)
        if block.element_size() == 1:
            return block.view(torch.uint8)[pages, head][:, at.reshape(-1)].view(pool.dtype).view(-1, D)
        return block[pages, head][:, at.reshape(-1)].view(-1, D)

    def keys(pages, head):
        shift_c = c.expand(PAGE, D).repeat(pages.shape[0], 1)
        if fmt == "q2":
            code = (element(pools["k_q"], pages, head, at_2).long() >> (2 * (shift_c & 3))) & 3
            k = code.double() * element(pools["k_scale"], pages, head, at_s).double()
            k = k + element(pools["k_zero"], pages, head, at_s).double()
        else:
            code = (element(pools["k"], pages, head, at_4).long() >> (4 * (shift_c & 1))) & 15
            per = 16 if fmt == "nvfp4" else 64
            s = element(pools["k_scale"], pages, head, t * (D // per) + c // per).double()
            if fmt == "nvfp4":
                mag = torch.tensor(_E2M1, dtype=torch.float64, device=dev)[code & 7]
                k = torch.where(code > 7, -mag, mag) * s
            else:  # the codebook's values are the 32-bit ones
                k = torch.tensor(_NF4, dtype=torch.float32, device=dev).double()[code] * s
        return k + element(pools["k_res"], pages, head, at_res).double()

    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    for i, (T, ql) in enumerate(zip(geo["lens"], geo["q"])):
        pages = st["table"][i, :-(-T // PAGE)].long()
        for h in range(H):
            k = keys(pages, h)[:T]
            v = element(pools["v"], pages, h, at_v).double()[:T]
            for r in range(G):
                for a in range(0, ql, 512):
                    e = min(a + 512, ql)
                    x = q[i, a:e, h * G + r].double()
                    s = x @ k.T / math.sqrt(D)
                    seen = torch.arange(T, device=dev)[None, :] <= torch.arange(T - ql + a, T - ql + e, device=dev)[:, None]
                    w = torch.softmax(s.masked_fill(~seen, -math.inf), dim=-1)
                    out[i, a:e, h * G + r] = w @ v
    return out
