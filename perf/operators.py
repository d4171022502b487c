"""What a decoder needs when it answers, as timed cases: a cache of keys and
values in 4 bits with the attention that reads it, and log probabilities by
token id with their gradient.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from
the seed alone, ``run`` is one pass, in elementary torch operations or, where
``own`` is true, by the C ABI's entry points on the same buffers.  ``exact``
gives the same results in float64, ``work`` the bytes and operations that a
pass cannot do without (each input read once, each output written once).

The cache holds groups of 32 neighbouring elements of a token's head row as
E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; two a byte, the even
element in the low nibble) that share one scale 2^e, held as the byte e + 127.
e is the smallest number with amax <= 6 * 2^e, at least -119; elements are
rounded to the nearest code, ties to the even one; a group of zeros has the
byte 127.  Codes lie as (page, head, token of the page, D/2) bytes, scales as
(page, head, token of the page, D/32), and page_table (sequence, place) says
which page holds a sequence's tokens from place * page_size on (-1: none).
Sequence b holds tokens 0 .. start[b] - 1 before the call, and the call's T
rows are its next ones, of which count[b] are valid (all T without count).
"""

from __future__ import annotations

import functools
import math

import torch

own = False


def listed():
    return [
        # One token of one request on a short context: latency decides.
        dict(name="attend_one", kind="attend", B=1, T=1, Hq=4, Hkv=4, D=64, L=256, page=16, causal=True, ragged=False),
        # A serving batch, one token each, four query heads to a cached head, contexts of all lengths.
        dict(name="attend_batch", kind="attend", B=32, T=1, Hq=32, Hkv=8, D=128, L=8192, page=64, causal=True, ragged=False),
        # Few requests on long contexts, every head with keys of its own.
        dict(name="attend_long", kind="attend", B=4, T=1, Hq=16, Hkv=16, D=128, L=32768, page=256, causal=True, ragged=False),
        # Drafted tokens checked in one pass: a few rows each, padded to the longest draft.
        dict(name="attend_drafts", kind="attend", B=16, T=5, Hq=16, Hkv=16, D=64, L=3001, page=32, causal=True, ragged=True),
        # A long prompt read piece by piece: a thousand new rows on what is cached.
        dict(name="attend_chunk", kind="attend", B=2, T=1024, Hq=32, Hkv=8, D=128, L=8192, page=64, causal=True, ragged=False),
        # A step of a serving batch: one token each goes into the cache, and is read back.
        dict(name="store_step", kind="store", B=64, T=1, Hkv=8, D=128, L=2048, page=64, ragged=False),
        # Prompts of different lengths, padded, written from the packed projection and read back.
        dict(name="store_prompts", kind="store", B=8, T=4096, Hkv=16, D=64, L=4096, page=32, ragged=True),
        # A cached context read back whole.
        dict(name="read_context", kind="read", B=4, T=8191, Hkv=8, D=128, L=8191, page=128, ragged=True),
        # A step's logits over a large vocabulary: the chosen tokens and their 20 best alternatives.
        dict(name="score_step", kind="score", rows=8, classes=131072, pad=0, top=20),
        # A prompt's tokens scored, with the five best alternatives of each; rows of an odd size, padded apart.
        dict(name="score_prompt", kind="score", rows=4096, classes=32001, pad=31, top=5),
        # The gradient of a small batch's log probabilities.
        dict(name="grad_small", kind="grad", rows=64, classes=1000, pad=0),
        # The same for a training batch over a vocabulary, entropy bonus included.
        dict(name="grad_train", kind="grad", rows=4096, classes=50021, pad=0),
    ]


# ---- drawn cases: the same ranges ----


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choices(("attend", "store", "read", "score", "grad"), weights=(6, 2, 1, 3, 2))[0]
    if kind == "score":
        classes = _log_int(rng, 10, 131072)
        return dict(kind=kind, rows=_log_int(rng, 1, min(4096, max(1, (1 << 27) // classes))), classes=classes,
                    pad=rng.choice((0, 0, rng.randint(1, 64))), top=min(classes, rng.choice((0, 1, 5, 20, rng.randint(1, 64)))))
    if kind == "grad":
        classes = _log_int(rng, 10, 131072)
        return dict(kind=kind, rows=_log_int(rng, 1, min(8192, max(1, (1 << 27) // classes))), classes=classes,
                    pad=rng.choice((0, 0, rng.randint(1, 64))))
    D, page, Hkv = rng.choice((32, 64, 128)), rng.choice((16, 32, 64, 128, 256)), rng.choice((1, 2, 4, 5, 8, 16))
    if kind == "attend":
        Hq = Hkv * rng.choice((1, 1, 2, 3, 4, 7, 8))
        T = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1024)
        L = max(T, _log_int(rng, 16, 32768))
        most = min((1 << 26) * 4 // (Hkv * L * D), (1 << 36) // (Hq * T * L * D))
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(64, most))), T=T, Hq=Hq, Hkv=Hkv, D=D, L=L, page=page,
                    causal=rng.random() < 0.8, ragged=rng.random() < 0.4)
    L = _log_int(rng, 16, 16384)
    T = L if kind == "read" else 1 if rng.random() < 0.4 else _log_int(rng, 2, L)
    B = _log_int(rng, 1, max(1, min(64, (1 << 25) // (L * Hkv * D))))
    return dict(kind=kind, B=B, T=T, Hkv=Hkv, D=D, L=L, page=page, ragged=rng.random() < 0.5)


# ---- inputs ----


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise(x):
    """Codes and scales of x (..., D): uint8 (..., D/2) and (..., D/32)."""
    group = x.unflatten(-1, (-1, 32))
    amax = group.abs().amax(-1, keepdim=True)
    # amax = f * 2^x with 1 <= f < 2: e is x - 2 where f <= 1.5, else x - 1.
    byte = (((amax.view(torch.int32) + 0x3FFFFF) >> 23) - 2).clamp(min=8)
    byte = torch.where(amax > 0, byte, torch.full_like(byte, 127))
    y = group.abs() * ((254 - byte) << 23).view(torch.float32)
    code = torch.where(y < 2, torch.round(2 * y), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4))
    code = (code.to(torch.uint8) | (torch.signbit(group).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte[..., 0].to(torch.uint8)


def _lengths(g, case):
    """start, count: sequence b's tokens before the call, and its new ones (None: T each)."""
    B, T, L = case["B"], case["T"], case["L"]
    count = torch.randint(1, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    start = (torch.rand((B,), generator=g, device="cuda") * (L - T + 1)).to(torch.int32).clamp(max=L - T)
    start[0] = L - T
    return start, count


def _pages(g, case):
    """A page table in which the sequences' pages are strewn, and the number of pages."""
    places = -(-case["L"] // case["page"])
    n = case["B"] * places
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32).reshape(case["B"], places), n


def prepare(case, seed):
    g, c = torch.Generator(device="cuda").manual_seed(int(seed)), case
    kind = c["kind"]
    if kind in ("score", "grad"):
        rows, classes = c["rows"], c["classes"]
        st = dict(kind=kind, top=c.get("top", 0), logits=(3 * _normal(g, rows, classes + c["pad"]))[:, :classes],
                  tokens=torch.randint(classes, (rows,), generator=g, device="cuda", dtype=torch.int32))
        if rows > 4:
            st["tokens"][3] = -1  # a padded place
        if kind == "grad":
            x = st["logits"].double()
            logp = torch.log_softmax(x, -1)
            st["lse"] = torch.logsumexp(x, -1).float()
            st["entropy"] = -(logp.exp() * logp).sum(-1).float()
            st["d_logp"], st["d_entropy"] = -torch.rand((rows,), generator=g, device="cuda"), 0.1 * _normal(g, rows)
        return st
    B, T, H, D, page = c["B"], c["T"], c["Hkv"], c["D"], c["page"]
    table, n = _pages(g, c)
    start, count = _lengths(g, c)
    # Keys' channels differ in size, as trained projections make them.
    spread = torch.exp(0.5 * _normal(g, H, 1, D))
    st = dict(kind=kind, table=table, start=start, count=count, page=page, T=T, D=D, H=H, L=c["L"])
    st["k_codes"], st["k_scales"] = _quantise(_normal(g, n, H, page, D) * spread)
    st["v_codes"], st["v_scales"] = _quantise(_normal(g, n, H, page, D))
    if kind == "attend":
        st["q"] = _normal(g, B, T, c["Hq"], D)
        st["scale"], st["causal"] = 1 / math.sqrt(D), c["causal"]
    if kind == "read":
        st["start"] = torch.zeros_like(start)
    if kind == "store":
        st["kv"] = _normal(g, B, T, 2, H, D)
        st["kv"][:, :, 0] *= spread.reshape(H, D)
    return st


# ---- the plain forms ----


@functools.cache
def _byte_pairs():
    """The two values of a byte of codes, (256, 2)."""
    value = [0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6]
    return torch.tensor([[value[b & 15], value[b >> 4]] for b in range(256)], device="cuda")


def _values(codes, scales):
    """What codes (..., D/2) and scales (..., D/32) stand for, (..., D)."""
    pairs = _byte_pairs()[codes.int()].flatten(-2)
    return (pairs.unflatten(-1, (-1, 32)) * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _gathered(st, name):
    """The cache's values in each sequence's order, (B, H, places * page, D)."""
    pages = st["table"].clamp(min=0)
    codes, scales = (st["%s_%s" % (name, part)][pages].transpose(1, 2).flatten(2, 3) for part in ("codes", "scales"))
    return _values(codes, scales)


def _new(st):
    """Which of the call's T rows are valid, (B, T), and their places in their sequences."""
    t = torch.arange(st["T"], device="cuda")
    at = st["start"][:, None] + t
    return torch.ones_like(at, dtype=torch.bool) if st["count"] is None else t < st["count"][:, None], at


def _plain_attend(st):
    q, H = st["q"], st["H"]
    B, T, Hq, D = q.shape
    valid, at = _new(st)
    k, v = _gathered(st, "k"), _gathered(st, "v")
    q = q.permute(0, 2, 1, 3).reshape(B, H, (Hq // H) * T, D)
    s = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (Hq // H, T)) * st["scale"]
    j = torch.arange(k.shape[2], device="cuda")
    last = at if st["causal"] else (st["start"] + (T if st["count"] is None else st["count"]))[:, None] - 1
    seen = (j <= last[..., None]).expand(B, T, -1) & valid[..., None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (Hq // H, T)) / total.clamp(min=1e-30)
    lse = torch.log(total) + m
    return o.flatten(1, 2).transpose(1, 2).contiguous(), lse[..., 0].flatten(1, 2)


def _plain_read(st):
    valid, at = _new(st)
    page = torch.gather(st["table"], 1, (at // st["page"]).clamp(max=st["table"].shape[1] - 1)).long()
    slot = at % st["page"]
    read = lambda n: _values(st[n + "_codes"][page, :, slot], st[n + "_scales"][page, :, slot]) * valid[..., None, None]  # noqa: E731
    return read("k"), read("v")


def _plain_store(st):
    valid, at = _new(st)
    b, t = valid.nonzero(as_tuple=True)
    at = at[b, t].long()
    page, slot = st["table"][b, at // st["page"]].long(), at % st["page"]
    kc, ks = _quantise(st["kv"][b, t, 0])
    vc, vs = _quantise(st["kv"][b, t, 1])
    st["k_codes"][page, :, slot], st["k_scales"][page, :, slot] = kc, ks
    st["v_codes"][page, :, slot], st["v_scales"][page, :, slot] = vc, vs
    return _plain_read(st)


def _chosen(x, tokens):
    valid = (tokens >= 0) & (tokens < x.shape[1])
    return valid, torch.gather(x, 1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0]


def _best(x, k):
    """The k largest of each row in order, ties to the lowest index: torch's own order of ties is not said, so keys carry the index."""
    bits = (x + 0.0).contiguous().view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key = key | (0xFFFFFFFF - torch.arange(x.shape[1], device="cuda"))
    return (0xFFFFFFFF - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)).to(torch.int32)


def _plain_score(st):
    x = st["logits"]
    m = x.amax(-1, keepdim=True)
    shifted = x - m
    e = torch.exp(shifted)
    total = e.sum(-1)
    log_total = torch.log(total)
    valid, at = _chosen(shifted, st["tokens"])
    logp = torch.where(valid, at - log_total, torch.zeros_like(at))
    out = dict(logp=logp, lse=m[:, 0] + log_total, entropy=log_total - (e * shifted).sum(-1) / total)
    if st["top"]:
        out["top"] = _best(x, st["top"])
        out["top_logp"] = torch.gather(shifted, 1, out["top"].long()) - log_total[:, None]
    return out


def _plain_grad(st):
    x = st["logits"]
    valid, _ = _chosen(x, st["tokens"])
    logp = x - st["lse"][:, None]
    d_logp = torch.where(valid, st["d_logp"], torch.zeros_like(st["d_logp"]))
    grad = -torch.exp(logp) * (d_logp[:, None] + st["d_entropy"][:, None] * (logp + st["entropy"][:, None]))
    return grad.scatter_add(1, st["tokens"].clamp(0, x.shape[1] - 1).long()[:, None], d_logp[:, None])


# ---- the framework's entry points ----


def _cache(st):
    from ember_amd import capi
    return capi.KVCacheView(st["k_codes"].data_ptr(), st["k_scales"].data_ptr(), st["v_codes"].data_ptr(), st["v_scales"].data_ptr(),
                            st["table"].data_ptr(), st["k_codes"].shape[0], st["H"], st["page"], st["D"], *st["table"].shape)


def _own_run(st):
    from ember_amd import capi
    L, kind = capi.lib(), st["kind"]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if kind in ("score", "grad"):
        x, tokens = st["logits"], st["tokens"].data_ptr()
        rows, classes = x.shape
    if kind == "score":
        k = st["top"]
        out = dict(logp=new(rows), lse=new(rows), entropy=new(rows))
        if k:
            out["top"], out["top_logp"] = new(rows, k, dtype=torch.int32), new(rows, k)
        at = [t.data_ptr() for t in out.values()]
        capi.check(L.token_logprobs(x.data_ptr(), x.stride(0), tokens, rows, classes, *at, *(() if k else (None, None)), k), "token_logprobs")
        return out
    if kind == "grad":
        grad = new(rows, classes)
        capi.check(L.token_logprobs_bwd(x.data_ptr(), x.stride(0), tokens, st["lse"].data_ptr(), st["entropy"].data_ptr(), st["d_logp"].data_ptr(),
                                        st["d_entropy"].data_ptr(), grad.data_ptr(), classes, rows, classes), "token_logprobs_bwd")
        return grad
    cache, T, H, D = _cache(st), st["T"], st["H"], st["D"]
    start, count = st["start"].data_ptr(), None if st["count"] is None else st["count"].data_ptr()
    B = st["table"].shape[0]
    if kind == "attend":
        Hq = st["q"].shape[2]
        o, lse = torch.empty_like(st["q"]), new(B, Hq, T)
        at = (T * Hq * D, D, Hq * D)
        capi.check(L.kv_cache_attention(cache, st["q"].data_ptr(), o.data_ptr(), lse.data_ptr(), T, Hq, st["scale"], int(st["causal"]),
                                        *at, *at, start, count), "kv_cache_attention")
        return o, lse
    if kind == "store":
        kv = st["kv"]
        capi.check(L.kv_cache_write(cache, kv.data_ptr(), kv[:, :, 1].data_ptr(), T, T * 2 * H * D, D, 2 * H * D, start, count, None), "kv_cache_write")
    k, v = new(B, T, H, D), new(B, T, H, D)
    capi.check(L.kv_cache_read(cache, k.data_ptr(), v.data_ptr(), T, T * H * D, D, H * D, start, count), "kv_cache_read")
    return k, v


def run(st):
    if own:
        return _own_run(st)
    return dict(attend=_plain_attend, store=_plain_store, read=_plain_read, score=_plain_score, grad=_plain_grad)[st["kind"]](st)


# ---- the same in float64 ----


def _exact_values(codes, scales):
    """Decoded from the bits: sign, two bits of exponent, one of fraction."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    sign, rest = 1 - 2 * torch.floor(n / 8), n % 8
    exponent, fraction = torch.floor(rest / 2), rest % 2
    size = torch.where(exponent > 0, (1 + fraction / 2) * 2.0 ** (exponent - 1), fraction / 2)
    return sign * size * torch.repeat_interleave(2.0 ** (scales.double() - 127), 32, -1)


def _exact_round(x):
    """x held in the cache: the nearest code by distance, of two as near the even one."""
    group = x.double().unflatten(-1, (-1, 32))
    amax = group.abs().amax(-1, keepdim=True)
    step = 2.0 ** torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 6)) / 6)).clamp(min=-119)
    size, grid = group.abs() / step, torch.tensor([0, 1, 2, 4, 0.5, 1.5, 3, 6], device="cuda", dtype=torch.float64)
    best, off = torch.zeros_like(size), size.clone()
    for value in grid[1:]:  # the even codes come first, so that an odd one has to be nearer
        d = (size - value).abs()
        best, off = torch.where(d < off, value, best), torch.minimum(d, off)
    return (torch.sign(group) * best * step).flatten(-2)


def _sequence(st, name, b, n):
    """Sequence b's first n tokens, (H, n, D)."""
    pages = st["table"][b, :-(-n // st["page"])].long()
    codes, scales = (st["%s_%s" % (name, part)][pages] for part in ("codes", "scales"))
    return _exact_values(codes, scales).transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_attend(st):
    q, H = st["q"].double(), st["H"]
    B, T, Hq, D = q.shape
    o, lse = torch.zeros_like(q), torch.full((B, Hq, T), -math.inf, device="cuda", dtype=torch.float64)
    for b in range(B):
        n = T if st["count"] is None else int(st["count"][b])
        first = int(st["start"][b])
        k, v = _sequence(st, "k", b, first + n), _sequence(st, "v", b, first + n)
        for h in range(Hq):
            s = torch.matmul(q[b, :n, h], k[h // (Hq // H)].t().contiguous()) * st["scale"]
            if st["causal"]:
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(first + 1), -math.inf)
            lse[b, h, :n] = torch.logsumexp(s, -1)
            o[b, :n, h] = torch.matmul(torch.softmax(s, -1), v[h // (Hq // H)])
    return o, lse


def exact(case, seed):
    st = prepare(case, seed)
    kind = st["kind"]
    if kind == "attend":
        return _exact_attend(st)
    if kind in ("store", "read"):
        if kind == "store":
            out = [_exact_round(st["kv"][:, :, i]) for i in (0, 1)]
        else:  # one sequence after the other
            B, T = st["table"].shape[0], st["T"]
            out = [torch.stack([_sequence(st, n, b, T).transpose(0, 1) for b in range(B)]) for n in ("k", "v")]
        if st["count"] is not None:
            for b, n in enumerate(st["count"].tolist()):
                out[0][b, n:], out[1][b, n:] = 0, 0
        return out[0], out[1]
    x, tokens = st["logits"].double(), st["tokens"].long()
    rows = torch.arange(x.shape[0], device="cuda")
    known = (tokens >= 0) & (tokens < x.shape[1])
    if kind == "score":
        logp = torch.log_softmax(x, -1)
        out = dict(logp=torch.where(known, logp[rows, tokens.clamp(min=0)], 0.0), lse=torch.logsumexp(x, -1),
                   entropy=-(logp.exp() * logp).sum(-1))
        if st["top"]:
            order = torch.stack([torch.sort(r, descending=True, stable=True).indices[:st["top"]] for r in x])
            out["top"], out["top_logp"] = order.to(torch.int32), torch.gather(logp, 1, order)
        return out
    # From the lse and the entropy that the call is given, as they are.
    logp = x - st["lse"].double()[:, None]
    d_logp, d_entropy = st["d_logp"].double() * known, st["d_entropy"].double()
    grad = -logp.exp() * (d_logp + d_entropy * st["entropy"].double())[:, None] - d_entropy[:, None] * logp.exp() * logp
    grad[rows, tokens.clamp(min=0)] += d_logp
    return grad


# ---- what a pass cannot do without ----


def work(case):
    c, kind = case, case["kind"]
    if kind in ("score", "grad"):
        n = c["rows"] * c["classes"]
        if kind == "score":
            return dict(bytes=4 * n + 4 * c["rows"] * (4 + 2 * c["top"]), flops=6 * n)
        return dict(bytes=8 * n + 20 * c["rows"], flops=8 * n)
    row = 2 * c["Hkv"] * c["D"]  # a token's keys and values
    new = c["B"] * c["T"] * (0.5 if c["ragged"] else 1)  # valid rows, on average
    if kind == "attend":
        # start is spread evenly over 0 .. L - T, the first sequence's is L - T.
        held = c["B"] * c["T"] * (0.5 if c["ragged"] else 1) + (c["L"] - c["T"]) * (1 + c["B"]) / 2
        seen = held / c["B"] - (new / c["B"] / 2 if c["causal"] else 0)
        return dict(bytes=held * row * 17 / 32 + 8 * c["B"] * c["T"] * c["Hq"] * c["D"], flops=4 * new * c["Hq"] * seen * c["D"])
    out = 4 * c["B"] * c["T"] * row
    if kind == "read":
        return dict(bytes=new * row * 17 / 32 + out, flops=new * row)
    return dict(bytes=new * row * (4 + 17 / 16) + out, flops=8 * new * row)
