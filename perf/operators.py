"""The operators of a serving step over many sessions, as cases that can be timed and checked: the
KV cache held in 8 bits (written, read back, attended), decode attention of a batch whose streams
share a long prefix, and the log probabilities of the tokens picked.

Sizes are the Qwen3-ASR text decoder's attention (16 query / 8 KV heads of 128) and vocabulary
(151936), as the tests and the benchmark use them, from one stream to a server's batch, contexts
of tens to some thousands of keys.

The 8-bit cache, as the library lays it out: pages of `ps` positions (a multiple of 16); K codes
[page, Hkv, ps, Dh], V codes in blocks of 16 positions with the dims outside, [page, Hkv, ps / 16,
Dh, 16], one fp32 scale per position and head, [page, Hkv, ps], for each of K and V."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HQ, HKV, DH = 16, 8, 128
G = HQ // HKV
VOCAB = 151936
SCALE = 1.0 / math.sqrt(DH)
TINY = 2.0 ** -126


def listed():
    return [
        # one decode step's new K/V rows of a full batch going into the 8-bit cache, and read back:
        # the smallest call, latency only
        {"name": "cache_step_16", "kind": "cache", "B": 16, "T": 1, "L": 1000, "ps": 16,
         "out": "float32"},
        # the longest prompt the decoder's default context takes, written after a first turn
        {"name": "cache_prompt_2048", "kind": "cache", "B": 1, "T": 2048, "L": 2700, "ps": 64,
         "out": "float32"},
        # a few sessions' contexts read back as bf16, as the prompt attention takes them
        {"name": "cache_read_717", "kind": "cache_read", "B": 4, "T": 717, "ps": 32,
         "out": "bfloat16"},
        # a server's sessions read back in fp32
        {"name": "cache_read_4096", "kind": "cache_read", "B": 16, "T": 4096, "ps": 16,
         "out": "float32"},
        # a single transcription's decode attention over the 8-bit cache: latency
        {"name": "decode_q8_one", "kind": "decode", "B": 1, "L": 1301, "ps": 16},
        # a few live streams of different lengths
        {"name": "decode_q8_few", "kind": "decode", "B": 6, "L": 1101, "ps": 16},
        # a server's full batch over long contexts: the HBM-bound end
        {"name": "decode_q8_many", "kind": "decode", "B": 16, "L": 4097, "ps": 16},
        # a few sessions behind one prompt, the bf16 cache
        {"name": "shared_few", "kind": "shared", "B": 6, "P": 503, "own": 64, "ps": 16, "q8": False},
        # a full batch behind a long prompt, the 8-bit cache
        {"name": "shared_q8_16", "kind": "shared", "B": 16, "P": 2048, "own": 257, "ps": 64,
         "q8": True},
        # a large batch behind the longest prompt, the bf16 cache
        {"name": "shared_many", "kind": "shared", "B": 64, "P": 4096, "own": 512, "ps": 16,
         "q8": False},
        # the confidence of one greedy step's token with its five best alternatives
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "top": 5},
        # a transcript's tokens scored in one pass
        {"name": "logprobs_257", "kind": "logprobs", "rows": 257, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("cache", "cache_read", "decode", "decode", "shared", "shared", "logprobs"))
    ps = rng.choice((16, 32, 64, 128))
    out = rng.choice(("float32", "bfloat16"))
    if kind == "cache":
        if rng.random() < 0.5:
            return {"kind": kind, "B": _log(rng, 1, 64), "T": 1, "L": _log(rng, 64, 4096),
                    "ps": ps, "out": out}
        T = _log(rng, 2, 2048)
        return {"kind": kind, "B": rng.randint(1, 4), "T": T, "L": T + rng.randint(1, 2000),
                "ps": ps, "out": out}
    if kind == "cache_read":
        return {"kind": kind, "B": rng.randint(1, 16), "T": _log(rng, 16, 4096), "ps": ps,
                "out": out}
    if kind == "decode":
        return {"kind": kind, "B": _log(rng, 1, 16), "L": _log(rng, 40, 4096) + 1, "ps": ps}
    if kind == "shared":
        return {"kind": kind, "B": _log(rng, 2, 64), "P": _log(rng, 64, 4096),
                "own": _log(rng, 8, 512), "ps": ps, "q8": rng.random() < 0.5}
    return {"kind": kind, "rows": _log(rng, 1, 256), "top": rng.randint(1, 20)}


# ------------------------------------------------------------------------- inputs ----
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) + 1)


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV).mul_(std)


def _lengths(g, B, L, lo):
    """Positions each stream holds: the longest L, the others from `lo` up."""
    r = torch.randint(lo, L + 1, (B,), generator=g, device=DEV)
    r[0] = L
    return r


def _table(g, B, pages):
    return torch.randperm(B * pages, generator=g, device=DEV).reshape(B, pages).to(torch.int32)


def _pool_q8(g, n_pages, ps):
    """K and V codes and scales of random rows, in the library's layout."""
    st = {}
    for name in ("k", "v"):
        x = _randn(g, n_pages, HKV, ps, DH)
        s = x.abs().amax(-1) / 127
        c = torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8)
        if name == "v":
            c = c.reshape(n_pages, HKV, ps // 16, 16, DH).transpose(3, 4).contiguous()
        st[name + "q"], st[name + "s"] = c, s
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["p"] = {n: t.data_ptr() for n, t in st.items() if isinstance(t, torch.Tensor)}
    return st


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "logprobs":
        rows = case["rows"]
        x = _randn(g, rows, VOCAB, std=2.5)
        # a few likely tokens stand out, and some ids are banned
        at = torch.randint(0, VOCAB, (rows, 12), generator=g, device=DEV)
        x.scatter_add_(1, at, _randn(g, rows, 12).abs_().mul_(6.0))
        x[:, torch.randint(0, VOCAB, (64,), generator=g, device=DEV)] = -math.inf
        pick = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, x.argmax(1),
                           torch.randint(0, VOCAB, (rows,), generator=g, device=DEV))
        return {"case": case, "x": x, "tokens": pick.to(torch.int32),
                "logprob": torch.empty(rows, device=DEV), "entropy": torch.empty(rows, device=DEV),
                "ids": torch.empty(rows, case["top"], dtype=torch.int32, device=DEV),
                "top": torch.empty(rows, case["top"], device=DEV)}
    B, ps = case["B"], case["ps"]
    if kind in ("cache", "cache_read"):
        T = case["T"]
        L = case["L"] if kind == "cache" else T
        pages = -(-(L + 8) // ps)
        st = {"case": case, "table": _table(g, B, pages), "pages": pages, "n_pages": B * pages}
        if kind == "cache":
            st["pos"] = (_lengths(g, B, L, T) - T).to(torch.int32)
            st["k"] = _randn(g, B, T, HKV, DH)
            st["v"] = _randn(g, B, T, HKV, DH)
            n = st["n_pages"]
            st["kq"] = torch.zeros(n, HKV, ps, DH, dtype=torch.int8, device=DEV)
            st["vq"] = torch.zeros(n, HKV, ps // 16, DH, 16, dtype=torch.int8, device=DEV)
            st["ks"] = torch.zeros(n, HKV, ps, device=DEV)
            st["vs"] = torch.zeros(n, HKV, ps, device=DEV)
        else:
            st["pos"] = torch.zeros(B, dtype=torch.int32, device=DEV)
            st.update(_pool_q8(g, st["n_pages"], ps))
        dt = getattr(torch, case["out"])
        st["ko"] = torch.empty(B, T, HKV, DH, dtype=dt, device=DEV)
        st["vo"] = torch.empty(B, T, HKV, DH, dtype=dt, device=DEV)
        return st
    if kind == "decode":
        L, P = case["L"], 0
        lens = _lengths(g, B, L, max(1, L // 2))
    else:
        P = case["P"]
        L = P + case["own"]
        lens = _lengths(g, B, L, P + 1)
    pages = -(-(L + 64) // ps)  # room for the tokens still to come
    table = _table(g, B, pages)
    table[:, :P // ps] = table[0, :P // ps]
    st = {"case": case, "table": table, "pages": pages, "n_pages": B * pages, "P": P,
          "pos": (lens - 1).to(torch.int32), "q": _randn(g, B, HQ, DH, std=2.0),
          "out": torch.empty(B, HQ, DH, device=DEV)}
    if case.get("q8", True):
        st.update(_pool_q8(g, st["n_pages"], ps))
    else:
        for name in ("kpool", "vpool"):
            st[name] = _randn(g, st["n_pages"], ps, HKV, DH).to(torch.bfloat16)
    if P % ps:  # the page that the prefix ends in: each stream has its own copy of its head
        i, r = P // ps, P % ps
        src, dst = table[0, i].long(), table[1:, i].long()
        for name in ("kpool", "vpool"):
            if name in st:
                st[name][dst, :r] = st[name][src, :r].clone()
        if "kq" in st:
            for name in ("kq", "ks", "vs"):
                st[name][dst, :, :r] = st[name][src, :, :r].clone()
            v = st["vq"].transpose(3, 4).reshape(-1, HKV, ps, DH)
            v[dst, :, :r] = v[src, :, :r].clone()
            st["vq"] = v.reshape(-1, HKV, ps // 16, 16, DH).transpose(3, 4).contiguous()
    return st


# ----------------------------------------------------------------------- plain form ----
def _where(st, pos):
    """(page, row in the page) of positions pos [B, n]; positions past the table's are not used."""
    ps = st["case"]["ps"]
    i = (pos // ps).clamp_(max=st["pages"] - 1)
    return torch.gather(st["table"].long(), 1, i), pos % ps


def _values(st, page, row):
    """K and V values [B, n, Hkv, Dh] in fp32 at (page, row)."""
    if "kpool" in st:
        return st["kpool"][page, row].float(), st["vpool"][page, row].float()
    k = st["kq"][page, :, row].float() * st["ks"][page, :, row][..., None]
    v = st["vq"][page, :, row // 16, :, row % 16].float() * st["vs"][page, :, row][..., None]
    return k, v


def _quantise(x):
    """Codes and scales of rows x [..., Dh]; the quotient in 64 bits, so that values next to the
    border of two codes go to the nearer one."""
    s = x.abs().amax(-1) / 127
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    d = torch.where(s > 0, s, torch.ones_like(s)).double()[..., None]
    c = torch.round(x.double() / d).clamp_(-127, 127)
    return torch.where(s[..., None] > 0, c, torch.zeros_like(c)).to(torch.int8), s


def _plain_cache(st):
    case = st["case"]
    n = st["pos"].long()[:, None] + torch.arange(case["T"], device=DEV)
    page, row = _where(st, n)
    if case["kind"] == "cache":
        c, s = _quantise(st["k"])
        st["kq"][page, :, row], st["ks"][page, :, row] = c, s
        c, s = _quantise(st["v"])
        st["vq"][page, :, row // 16, :, row % 16], st["vs"][page, :, row] = c, s
    k, v = _values(st, page, row)
    dt = getattr(torch, case["out"])
    return {"k": k.to(dt), "v": v.to(dt)}


def _plain_attention(st):
    lens = st["pos"].long() + 1
    L = st["case"]["L"] if st["case"]["kind"] == "decode" else st["P"] + st["case"]["own"]
    j = torch.arange(L, device=DEV)
    k, v = _values(st, *_where(st, j.expand(lens.numel(), -1).clone()))
    B = lens.numel()
    q = st["q"].reshape(B, HKV, G, DH)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * SCALE  # [B, Hkv, G, L]
    s = s.masked_fill(j >= lens[:, None, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v.transpose(1, 2).contiguous()) / p.sum(-1, keepdim=True)
    return o.reshape(B, HQ, DH)


def _plain_logprobs(st):
    x = st["x"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    weighted = (e * torch.where(e > 0, x - m, torch.zeros_like(x))).sum(1, keepdim=True)
    logprob = x.gather(1, st["tokens"].long()[:, None]) - lse
    # the order of the values with the lowest index first among equal ones, as one whole number
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -2147483648 - bits, bits)
    key = bits * (1 << 20) - torch.arange(VOCAB, device=DEV)
    ids = torch.topk(key, st["case"]["top"], dim=1).indices
    return {"logprob": logprob[:, 0], "entropy": (torch.log(total) - weighted / total)[:, 0],
            "ids": ids.to(torch.int32), "top": x.gather(1, ids) - lse}


# ------------------------------------------------------------------ the library's calls ----
def _own_run(st):
    from orator_amd import asr_ops, decoder_attn
    case = st["case"]
    kind = case["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    p = st["p"]
    if kind == "logprobs":
        asr_ops.TokenLogprobs(p["x"], VOCAB, p["tokens"], case["rows"], VOCAB, case["top"],
                              p["logprob"], p["entropy"], p["ids"], p["top"], stream)
        return {n: st[n] for n in ("logprob", "entropy", "ids", "top")}
    B, ps = case["B"], case["ps"]
    if kind in ("cache", "cache_read"):
        T = case["T"]
        if kind == "cache":
            decoder_attn.WriteKvCacheQ8Paged(p["k"], p["v"], HKV * DH, p["kq"], p["ks"], p["vq"],
                                             p["vs"], p["table"], st["pages"], ps, st["n_pages"], B,
                                             T, HKV, DH, p["pos"], stream)
        decoder_attn.ReadKvCacheQ8Paged(p["kq"], p["ks"], p["vq"], p["vs"], p["table"],
                                        st["pages"], ps, st["n_pages"], p["ko"], p["vo"],
                                        case["out"] == "bfloat16", B, T, HKV, DH, p["pos"], stream)
        return {"k": st["ko"], "v": st["vo"]}
    if kind == "decode":
        decoder_attn.GqaDecodeAttnQ8Paged(p["q"], p["kq"], p["ks"], p["vq"], p["vs"], p["table"],
                                          st["pages"], ps, st["n_pages"], p["pos"], p["out"], B,
                                          HQ, HKV, DH, SCALE, stream)
    elif case["q8"]:
        decoder_attn.GqaDecodeAttnSharedQ8Paged(p["q"], p["kq"], p["ks"], p["vq"], p["vs"],
                                                p["table"], st["pages"], ps, st["n_pages"],
                                                p["pos"], st["P"], p["out"], B, HQ, HKV, DH, SCALE,
                                                stream)
    else:
        decoder_attn.GqaDecodeAttnSharedPaged(p["q"], p["kpool"], p["vpool"], p["table"],
                                              st["pages"], ps, st["n_pages"], p["pos"], st["P"],
                                              p["out"], B, HQ, HKV, DH, SCALE, stream)
    return st["out"]


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    if kind == "logprobs":
        return _plain_logprobs(state)
    if kind in ("cache", "cache_read"):
        return _plain_cache(state)
    return _plain_attention(state)


# ------------------------------------------------------------------------------ work ----
def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        n = case["rows"] * VOCAB
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    if kind in ("cache", "cache_read"):
        n = case["B"] * case["T"] * HKV * 2  # rows of K and of V
        e = 2 if case["out"] == "bfloat16" else 4
        back = DH + 4 + DH * e
        if kind == "cache":
            return {"bytes": n * (4 * DH + DH + 4 + back), "flops": 5 * n * DH}
        return {"bytes": n * back, "flops": n * DH}
    B = case["B"]
    row = HKV * 2 * (DH + 4 if case.get("q8", True) else 2 * DH)
    if kind == "decode":
        keys = case["L"] + (B - 1) * 0.75 * case["L"]  # the mean of the lengths drawn
        read = keys
    else:
        mine = case["own"] + (B - 1) * 0.5 * case["own"]
        read = case["P"] + mine
        keys = B * case["P"] + mine
    return {"bytes": read * row + 8 * B * HQ * DH, "flops": 4 * keys * HQ * DH}


# -------------------------------------------------------------- the same in 64 bits ----
def _exact_row(st, b, n):
    """K and V [n, Hkv, Dh] of stream b's first n positions, float64, by flat row numbers."""
    ps = st["case"]["ps"]
    j = torch.arange(n, device=DEV)
    page = st["table"][b].long()[j // ps]
    if "kpool" in st:
        flat = page * ps + j % ps
        return tuple(st[x].reshape(-1, HKV, DH)[flat].double() for x in ("kpool", "vpool"))
    heads = torch.arange(HKV, device=DEV)
    line = (page[:, None] * HKV + heads) * ps + (j % ps)[:, None]  # [n, Hkv] rows of [.., Dh]
    k = st["kq"].reshape(-1, DH)[line].double() * st["ks"].reshape(-1)[line].double()[..., None]
    codes = st["vq"].transpose(3, 4).reshape(-1, DH)
    v = codes[line].double() * st["vs"].reshape(-1)[line].double()[..., None]
    return k, v


def _exact_values(x):
    """What rows x [..., Dh] read back as: scale fl32(amax / 127), codes to the nearest integer."""
    s = (x.abs().amax(-1, keepdim=True) / 127).double()
    c = torch.where(s >= TINY, (x.double() / s.clamp_min(TINY)).round(), torch.zeros_like(x).double())
    return c.clamp(-127, 127) * s


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        x = st["x"].double()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        return {"logprob": logp.gather(1, st["tokens"].long()[:, None])[:, 0],
                "entropy": -(p * logp.masked_fill(p == 0, 0.0)).sum(1),
                "ids": ids.to(torch.int32), "top": logp.gather(1, ids)}
    if kind == "cache":
        return {"k": _exact_values(st["k"]), "v": _exact_values(st["v"])}
    if kind == "cache_read":
        kv = [_exact_row(st, b, case["T"]) for b in range(case["B"])]
        return {"k": torch.stack([x[0] for x in kv]), "v": torch.stack([x[1] for x in kv])}
    out = torch.empty(case["B"], HQ, DH, dtype=torch.float64, device=DEV)
    for b in range(case["B"]):
        k, v = _exact_row(st, b, int(st["pos"][b]) + 1)
        for h in range(HQ):
            w = torch.softmax(k[:, h // G] @ st["q"][b, h].double() * SCALE, 0)
            out[b, h] = w @ v[:, h // G]
    return out
