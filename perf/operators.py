"""Serving from a paged key / value cache, operator by operator, as cases that can be timed and compared.

A case is a plain dict; ``op`` names what a pass does:

  write    rows of k and v go into a cache that holds them in 8 bits, and are read back in the compute type
  read     a range of a stored sequence is read back (moving it elsewhere, a contiguous call on it)
  decode   one query row per head over a cache that holds 8 bits
  step     one turn of a generation loop on such a cache: append a token, decode, forget it again
  chunk    ``new`` tokens per sequence, already appended, attend over everything cached (chunked prefill)
  verify   drafted tokens: append them, attend, forget them again

``listed()`` holds cases of each; ``draw()`` gives others of the same ranges.  ``store`` is what the cache holds: "int8" or
"fp8" (e4m3) with one fp32 scale per row of k and of v, "" = the compute type itself.  ``ragged``: lengths of the sequences between
half of ``n`` and ``n`` and, for chunk, between one and ``new`` new tokens each.
"""
import math

import torch

own = False   # False: the plain form below; True: the framework's operators

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
STORES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}   # largest code
LEAST = 2.0 ** -119                   # rows whose largest value is below this hold zeros


def listed():
    return [
        # A token of a few short chats: nothing but latency.
        dict(name="step_short", op="step", b=4, h=16, hk=4, n=777, d=64, r=32, dtype="fp16", store="int8", page=64, ragged=True),
        # A token against long caches, four query heads per key head: the stream of 8-bit keys and values.
        dict(name="decode_long", op="decode", b=8, h=32, hk=8, n=32768, d=128, r=64, dtype="bf16", store="int8", page=256, ragged=False),
        # A token against medium caches, a key head for every query head, every feature rotated.
        dict(name="decode_heads", op="decode", b=3, h=32, hk=32, n=8192, d=128, r=128, dtype="bf16", store="fp8", page=128, ragged=True),
        # A few tokens behind a short prompt enter the cache.
        dict(name="write_few", op="write", b=2, hk=4, n=37, d=96, r=48, dtype="fp16", store="fp8", page=64),
        # A long prompt enters the cache.
        dict(name="write_prompt", op="write", b=1, hk=8, n=32768, d=128, r=64, dtype="bf16", store="int8", page=256),
        # A stored sequence leaves the cache, but for its first and last tokens.
        dict(name="read_long", op="read", hk=32, n=16384, start=100, stop=16301, d=128, r=64, dtype="bf16", store="int8", page=256),
        # Five drafted tokens of eight requests are verified.
        dict(name="verify_draft", op="verify", b=8, h=32, hk=8, n=2000, new=5, d=128, r=64, dtype="bf16", store="", page=256, ragged=True),
        # The last short piece of a long prompt.
        dict(name="chunk_tail", op="chunk", b=1, h=32, hk=8, n=32768, new=64, d=128, r=64, dtype="bf16", store="", page=256, ragged=False),
        # A piece of a long document: the largest, bound by its products.
        dict(name="chunk_long", op="chunk", b=1, h=32, hk=8, n=16384, new=2048, d=128, r=128, dtype="bf16", store="", page=256, ragged=False),
        # Requests that are at different places: some bring one token, others hundreds.
        dict(name="chunk_mixed", op="chunk", b=6, h=8, hk=8, n=3001, new=300, d=96, r=48, dtype="fp16", store="", page=64, ragged=True),
        # Chunked prefill of two long prompts into 8 bits.
        dict(name="chunk_int8", op="chunk", b=2, h=32, hk=8, n=8192, new=512, d=128, r=64, dtype="bf16", store="int8", page=256, ragged=False),
        # A small model's chunk behind a shared prefix, in 8 bits.
        dict(name="chunk_fp8_small", op="chunk", b=4, h=8, hk=2, n=1500, new=33, d=64, r=64, dtype="fp16", store="fp8", page=128, ragged=True),
    ]


# ---- more of the same ranges ------------------------------------------------------------------------------------

def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "step", "chunk", "chunk", "chunk", "verify"])
    d = rng.choice([64, 96, 128, 128])
    hk = rng.choice([1, 2, 4, 8, 8, 16, 32])
    case = dict(op=op, b=_log_int(rng, 1, 16), h=hk * rng.choice([g for g in (1, 1, 2, 4, 8) if hk * g <= 64]), hk=hk, n=_log_int(rng, 64, 32768), d=d,
                r=rng.choice([d, d // 2]), dtype=rng.choice(["bf16", "fp16"]), store=rng.choice(["int8", "fp8"]), page=rng.choice([64, 128, 256]),
                ragged=rng.random() < 0.6)
    if op in ("write", "read"):
        del case["h"], case["ragged"]
    if op == "write":
        case["b"], case["n"] = rng.randint(1, 4), _log_int(rng, 1, 32768)
    if op == "read":
        del case["b"]
        case["start"] = rng.randint(0, case["n"] // 2)
        case["stop"] = rng.randint(case["start"] + 1, case["n"])
    if op in ("chunk", "verify"):
        case["store"] = rng.choice(["", "int8", "fp8"])
        case["new"] = _log_int(rng, 1, 16) if op == "verify" else min(case["n"], _log_int(rng, 2, 2048))
    while work(case)["bytes"] > 5e8 or work(case)["flops"] > 7e11 or case.get("b", 1) * case.get("h", 1) * case["n"] * case.get("new", 1) > 1.1e9:
        big = "b" if case.get("b", 1) > 1 else "n" if case["n"] > 2048 else "new" if case.get("new", 1) > 256 else "hk"
        if big == "hk":
            case["hk"] = max(1, case["hk"] // 2)
            if "h" in case:
                case["h"] = max(case["hk"], case["h"] // 2)
        else:
            case[big] = max(1, case[big] // 2)
        if "new" in case:
            case["new"] = min(case["new"], case["n"])
        if op == "read":
            case["stop"] = min(case["stop"], case["n"])
            case["start"] = min(case["start"], case["stop"] - 1)
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """Everything that is random, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, b, hk, n, d, r = DTYPES[case["dtype"]], case.get("b", 1), case["hk"], case["n"], case["d"], case["r"]
    op, new = case["op"], 1 if case["op"] in ("decode", "step") else case.get("new", 0)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # keys have features that are larger than others, the same ones in every token
    k = (rand(b, hk, n, d) * torch.exp(0.4 * rand(1, hk, 1, d))).to(dt)
    x = dict(k=k, v=rand(b, hk, n, d).to(dt), lens=[n] * b, counts=[new] * b)
    if case.get("ragged"):
        x["lens"] = torch.randint((n + 1) // 2, n + 1, (b,), generator=g, device="cuda").tolist()
        if op == "verify":   # drafts are as long as each other; the caches are not
            x["lens"] = [max(ln, min(n, new)) for ln in x["lens"]]
        elif op == "chunk":
            x["counts"] = torch.randint(1, new + 1, (b,), generator=g, device="cuda").tolist()
            x["counts"] = [min(c, ln) for c, ln in zip(x["counts"], x["lens"])]
    if "h" in case:
        x["q"] = rand(b, case["h"], new, d).to(dt)
        # the phases of a trained module: frequencies 10000^(-c / r), learned offsets over their whole range
        pos = torch.arange(n + new, device="cuda", dtype=torch.float32)
        inv = 10000.0 ** -(torch.arange(r, device="cuda", dtype=torch.float32) / r)
        x["freqs"] = pos[:, None] * inv
        x["bias"] = -2 * math.pi * torch.rand(hk, r, generator=g, device="cuda")
        if op in ("step", "verify"):   # the tokens that a pass appends
            x["k_new"], x["v_new"] = rand(b, hk, new, d).to(dt), rand(b, hk, new, d).to(dt)
    x["order"] = torch.randperm(b * -(-(n + new) // case["page"]), generator=g, device="cuda")   # which page comes next
    return x


def prepare(case, seed):
    """What a serving program holds: a filled cache (the plain form: its pages, scales, page table and lengths as tensors), the
    new rows and the phase table of fixed weights."""
    x = _inputs(case, seed)
    b, hk, n, d, page = case.get("b", 1), case["hk"], case["n"], case["d"], case["page"]
    s = dict(case=case, lens=x["lens"], scale=d ** -0.5)
    for name in ("q", "k_new", "v_new"):
        if name in x:
            s[name] = x[name]
    if "h" in case:
        s["pos_emb"] = (x["freqs"], x["bias"])
        s["counts"] = torch.tensor(x["counts"], dtype=torch.int32, device="cuda")
    if case["op"] == "write":
        s["k"], s["v"] = x["k"], x["v"]
    longest = n + (x["q"].shape[2] if "q" in x else 0)
    if own:
        from pope_pytorch_b200 import PagedKVCache
        cache = PagedKVCache(b, hk, d, num_pages=x["order"].numel(), page_size=page, max_seq_len=longest, dtype=DTYPES[case["dtype"]],
                             store=STORES.get(case["store"]))
        cache.alloc.free = x["order"].tolist()
        if case["op"] != "write":
            for i, ln in enumerate(x["lens"]):
                cache.append_to(i, x["k"][i, :, :ln], x["v"][i, :, :ln])
        s["cache"] = cache
        return s
    width = -(-longest // page)
    s["table"] = x["order"].view(b, width)
    s["len"] = torch.tensor(x["lens"], device="cuda")
    for name in ("k", "v"):
        codes, scales = _quantise(x[name], case["store"]) if case["store"] else (x[name], None)
        s[name + "_pages"] = torch.zeros(b * width, hk, page, d, dtype=codes.dtype, device="cuda")
        s[name + "_scales"] = torch.zeros(b * width, hk, page, device="cuda") if case["store"] else None
        if case["op"] != "write":
            _put(s, name, codes, scales, torch.zeros_like(s["len"]))
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------

def _quantise(x, store):
    """(codes, scale of each row) of (..., d) values."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    small = top < LEAST
    scaled = x * (TOP[store] / top.masked_fill(small, 1.0))
    codes = scaled.round() if store == "int8" else scaled
    return codes.masked_fill(small, 0.0).to(STORES[store]), (top / TOP[store]).masked_fill(small, 0.0).squeeze(-1)


def _slots(s, at, count):
    """(page, row of the page) of the tokens at .. at + count of every sequence, (b, count) each."""
    page = s["case"]["page"]
    pos = at[:, None] + torch.arange(count, device="cuda")
    return s["table"].gather(1, pos // page), pos % page


def _put(s, name, codes, scales, at):
    """codes (b, hk, n, d) and scales (b, hk, n) of tokens at .. at + n go into the pages."""
    pages, rows = _slots(s, at, codes.shape[2])
    if codes.shape[2] == 0:
        return
    target = s[name + "_pages"]
    if target.dtype == torch.float8_e4m3fn:   # (moved as bytes)
        target, codes = target.view(torch.uint8), codes.view(torch.uint8)
    target[pages, :, rows] = codes.permute(0, 2, 1, 3)
    if scales is not None:
        s[name + "_scales"][pages, :, rows] = scales.permute(0, 2, 1)


def _fetch(s, name, count):
    """The first ``count`` rows of every sequence in fp32, (b, hk, count, d)."""
    pages, rows = _slots(s, torch.zeros_like(s["len"]), count)
    held = s[name + "_pages"]
    got = (held.view(torch.uint8)[pages, :, rows].view(held.dtype) if held.dtype == torch.float8_e4m3fn else held[pages, :, rows]).float()
    if s[name + "_scales"] is not None:
        got = got * s[name + "_scales"][pages, :, rows][..., None]
    return got.permute(0, 2, 1, 3)


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _attend(s, lens, counts):
    """Rows i < counts[b] of q at positions lens[b] - counts[b] + i over the keys up to their own position."""
    case, (freqs, bias), q = s["case"], s["pos_emb"], s["q"]
    b, h, new, d = q.shape
    r, hk, n = case["r"], case["hk"], max(s["lens"]) + (new if case["op"] in ("step", "verify") else 0)
    k, v = _fetch(s, "k", n), _fetch(s, "v", n)
    row, key = torch.arange(new, device="cuda"), torch.arange(n, device="cuda")
    pos = (lens - counts)[:, None] + row                                    # (b, new)
    live = (row < counts[:, None]) & (pos >= 0)
    fq = freqs[pos.clamp(min=0)].double()[:, None]                          # (b, 1, new, r)
    fk = freqs[:n].double() + bias.double()[:, None]                        # (hk, n, r): angles in 64 bits
    q = q.float()
    aq, ak = _softplus(q[..., :r]), _softplus(k[..., :r])
    qe = torch.cat((aq * fq.cos().float(), aq * fq.sin().float(), q[..., r:]), -1)
    ke = torch.cat((ak * fk.cos().float(), ak * fk.sin().float(), k[..., r:]), -1)
    qe = qe.view(b, h // hk, hk, new, d + r).transpose(1, 2).reshape(b, hk, -1, d + r)   # query head g * hk + i reads key head i
    score = (qe @ ke.transpose(-1, -2) * s["scale"]).view(b, hk, h // hk, new, n)
    seen = (key <= pos[..., None]) & live[..., None]                        # (b, new, n)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    held = (key < lens[:, None])[:, None, :, None]
    out = p.reshape(b, hk, -1, n) @ v.masked_fill(~held, 0.0)
    out = out.view(b, hk, h // hk, new, d) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.transpose(1, 2).reshape(b, h, new, d).to(s["q"].dtype)


def _run_plain(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    op = case["op"]
    if op == "write":
        for name in ("k", "v"):
            _put(s, name, *_quantise(s[name], case["store"]), torch.zeros_like(s["len"]))
        return [[_fetch(s, name, case["n"])[i].to(dt) for name in ("k", "v")] for i in range(case["b"])]
    if op == "read":
        return [_fetch(s, name, case["stop"])[0, :, case["start"]:].to(dt) for name in ("k", "v")]
    lens, counts = s["len"], s["counts"].long()
    if op in ("step", "verify"):
        for name in ("k", "v"):
            x = s[name + "_new"]
            _put(s, name, *(_quantise(x, case["store"]) if case["store"] else (x, None)), lens)
        lens = lens + s["q"].shape[2]
    return _attend(s, lens, counts)


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    if not own:
        with torch.no_grad():
            return _run_plain(s)
    case, cache = s["case"], s["cache"]
    op = case["op"]
    if op == "write":
        cache.append(s["k"], s["v"])
        got = [cache.read(i) for i in range(case["b"])]
        cache.rollback(case["n"])
        return got
    if op == "read":
        return cache.read(0, case["start"], case["stop"])
    if op == "decode":
        return cache.decode(s["q"], s["pos_emb"], s["scale"])
    if op == "step":
        cache.append(s["k_new"], s["v_new"])
        out = cache.decode(s["q"], s["pos_emb"], s["scale"])
        cache.rollback(1)
        return out
    if op == "verify":
        cache.append(s["k_new"], s["v_new"])
        out = cache.attend(s["q"], s["pos_emb"], softmax_scale=s["scale"])
        cache.rollback(case["new"])
        return out
    return cache.attend(s["q"], s["pos_emb"], counts=s["counts"] if case["ragged"] else None, softmax_scale=s["scale"])


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------

def _held(x, store):
    """The values that a row's codes stand for, in 64 bits."""
    x = x.double()
    if not store:
        return x
    top = x.abs().max(dim=-1, keepdim=True).values
    y = torch.where(top < LEAST, torch.zeros_like(x), x / top * TOP[store])
    if store == "int8":
        y = torch.round(y)
    else:   # three bits behind the leading one, down to 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / step) * step
    return y * (top / TOP[store])


def exact(case, seed):
    x = _inputs(case, seed)
    op, store, r = case["op"], case["store"], case["r"]
    if op in ("write", "read"):
        lo, hi = case.get("start", 0), case.get("stop", case["n"])
        both = [_held(x[name], store)[:, :, lo:hi] for name in ("k", "v")]
        return [[t[i] for t in both] for i in range(case["b"])] if op == "write" else [t[0] for t in both]
    b, h, new, _ = x["q"].shape
    hk, out = case["hk"], torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        n, m = x["lens"][i], x["counts"][i]
        for e in range(hk):
            k, v = x["k"][i, e, :n], x["v"][i, e, :n]
            if op in ("step", "verify"):
                k, v = torch.cat((k, x["k_new"][i, e])), torch.cat((v, x["v_new"][i, e]))
            k, v = _held(k, store), _held(v, store)
            total = k.shape[0]
            angle = x["freqs"][:total].double() + x["bias"][e].double()
            mag = torch.logaddexp(k[:, :r], torch.zeros((), dtype=torch.float64, device="cuda"))
            kc, ks, kp = mag * torch.cos(angle), mag * torch.sin(angle), k[:, r:]
            mine = x["q"][i, e::hk, :m].double()                             # (heads of the group, m, d)
            at = torch.arange(total - m, total, device="cuda")
            f = x["freqs"][at].double()
            mag = torch.logaddexp(mine[..., :r], torch.zeros((), dtype=torch.float64, device="cuda"))
            dots = (mag * torch.cos(f)) @ kc.T + (mag * torch.sin(f)) @ ks.T + mine[..., r:] @ kp.T
            dots = dots * case["d"] ** -0.5
            later = torch.arange(total, device="cuda") > at[:, None]
            out[i, e::hk, :m] = torch.softmax(dots.masked_fill(later, -math.inf), -1) @ v
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; a multiply and an add for every product with a visible key (transcendental and
    elementwise work counts zero).  Ragged lengths are three quarters of ``n`` on average, ragged chunks half of ``new``."""
    op, hk, n, d, r = (case[x] for x in ("op", "hk", "n", "d", "r"))
    row = 2 * hk * ((d + 4) if case["store"] else 2 * d)     # a cached token, k and v
    if op == "write":   # tokens in, codes and scales out; those in, values out
        return dict(bytes=case["b"] * n * (2 * row + 2 * 4 * hk * d), flops=0)
    if op == "read":
        return dict(bytes=(case["stop"] - case["start"]) * (row + 4 * hk * d), flops=0)
    b, h, ragged = case["b"], case["h"], case["ragged"]
    new = 1 if op in ("decode", "step") else case["new"]
    kept = 0.75 * n if ragged else n
    rows = (new + 1) / 2 if ragged and op == "chunk" else new
    appended = new if op in ("step", "verify") else 0
    seen = kept + appended
    pairs = b * h * rows * max(1.0, seen - (rows - 1) / 2)
    return dict(bytes=b * (seen * row + appended * (row + 4 * hk * d) + 2 * 2 * h * rows * d) + 4 * n * r + 4 * hk * r, flops=2 * pairs * (2 * d + r))
