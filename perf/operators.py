"""Measured cases of the serving-step operators over the paged latent cache.

One decode or prefill step around the attention operators: where the step's
new rows go (block tables and slot maps), rotary positions, the latent-cache
writer and attention for a batch whose requests share one long prefix.  Each
operator has a plain form in elementary torch operations (`own` false), the
framework's call (`own` true) and a definition in 64 bits (`exact`).
"""
import math

import numpy as np
import torch

own = False

PAGE = 64      # rows per cache page
DC, DP = 512, 64   # latent and rotary width of a cache row
SM_SCALE = 1.0 / math.sqrt(192.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 requests: the call sits in front of every step, latency only
        dict(name="layout decode", op="layout", requests=64, most=1, rows=64, context=65536, prefix=0),
        # decode requests mixed with prefill chunks of a shared-prompt batch, outputs padded for a captured graph
        dict(name="layout mixed", op="layout", requests=509, most=4096, rows=32768, context=32768, prefix=2048),
        # the rotary slice of 64 decode queries, a strided view of 192-wide heads
        dict(name="rope decode", op="rope", rows=64, heads=16, width=64, offset=0, rot=64, pitch=192,
             layout="interleaved", dtype="bf16", inverse=False, base=10000.0, factor=40.0),
        # index queries of a prefill chunk: 64 of 128 dimensions rotated
        dict(name="rope index prefill", op="rope", rows=4096, heads=64, width=128, offset=0, rot=64, pitch=128,
             layout="half", dtype="bf16", inverse=False, base=10000.0, factor=40.0),
        # whole queries before absorption, last 64 of 192 rotated back, odd row count, 32-bit values
        dict(name="rope inverse fp32", op="rope", rows=1003, heads=128, width=192, offset=128, rot=64, pitch=192,
             layout="interleaved", dtype="fp32", inverse=True, base=500000.0, factor=1.0),
        # the new cache rows of a decode step
        dict(name="append decode", op="append", rows=64, pages=64, pitch=576, dtype="bf16", layout="interleaved", skip=0),
        # the cache rows of a prefill batch, read out of a wider projection, a few padded rows
        dict(name="append prefill", op="append", rows=16384, pages=300, pitch=2112, dtype="bf16", layout="interleaved", skip=37),
        # a single token after a short prompt: latency
        dict(name="prefix single", op="prefix", tokens=1, per=1, heads=16, prefix=1000, own=17),
        # decode of 64 requests behind a long document
        dict(name="prefix decode", op="prefix", tokens=64, per=1, heads=16, prefix=32768, own=512),
        # speculative decode, two tokens a request, own parts of ragged lengths, a prompt that ends inside a page
        dict(name="prefix ragged", op="prefix", tokens=256, per=2, heads=16, prefix=8001, own=1500),
        # all 128 heads on one GPU, few tokens, the longest context
        dict(name="prefix long", op="prefix", tokens=8, per=1, heads=128, prefix=131072, own=4096),
        # all 128 heads, a large batch: the tensor cores' case
        dict(name="prefix large", op="prefix", tokens=128, per=1, heads=128, prefix=16384, own=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("layout", "rope", "append", "prefix", "prefix"))
    if op == "layout":
        requests = _log(rng, 1, 512)
        most = _log(rng, 1, 4096)
        return dict(op=op, requests=requests, most=most, rows=min(32768, requests * most + rng.randrange(64)),
                    context=_log(rng, 1, 65536), prefix=rng.choice((0, _log(rng, 1, 131072))))
    if op == "rope":
        rot = rng.choice((32, 64, 64, 128))
        width = rot + rng.choice((0, 0, 64, 128))
        heads = _log(rng, 1, 128)
        return dict(op=op, rows=_log(rng, 1, max(1, (1 << 25) // (heads * width))) if heads * width > 64 else _log(rng, 1, 4096),
                    heads=heads, width=width, offset=rng.choice((0, width - rot)), rot=rot, pitch=width + rng.choice((0, 0, 64)),
                    layout=rng.choice(("interleaved", "half")), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    inverse=rng.random() < 0.3, base=rng.choice((10000.0, 500000.0)), factor=rng.choice((1.0, 4.0, 40.0)))
    if op == "append":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, pages=-(-rows // PAGE) + rng.randrange(1, 40), pitch=rng.choice((576, 576, 2112)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), layout=rng.choice(("interleaved", "half")),
                    skip=rng.randrange(min(rows, 50)))
    heads = rng.choice((16, 16, 16, 32, 48, 64, 128))
    per = rng.choice((1, 1, 2, 3))
    tokens = per * _log(rng, 1, 4096 // heads // per)
    prefix = _log(rng, 1, max(64, min(131072, (1 << 28) // (tokens * heads))))
    return dict(op=op, tokens=tokens, per=per, heads=heads, prefix=prefix, own=_log(rng, 1, min(4096, max(2, (1 << 18) // tokens))))


def _inv_freq(rot, base, factor, original=4096, fast=32.0, slow=1.0):
    """Inverse frequencies in 64 bits; factor > 1 stretches them for long contexts by parts (YaRN)."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    inv = base ** (-i / rot)
    if factor == 1.0:
        return inv
    at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return inv * (1 - ramp) + inv / factor * ramp


def _most_new(case):
    return max(1, min(case["most"], case["rows"]))


def _query_lens(case, host):
    """New rows of each request: mostly one, some chunks, some idle; never more than the outputs hold."""
    n, most = case["requests"], case["most"]
    q = np.ones(n, np.int64)
    if most > 1:
        chunk = host.random(n) < 0.05
        chunk[0] = True
        q[chunk] = np.exp(host.uniform(0, math.log(most), chunk.sum())).astype(np.int64)
        q[host.random(n) < 0.05] = 0
    return np.minimum(q, np.maximum(0, case["rows"] - np.concatenate([[0], np.cumsum(q)[:-1]]))).astype(np.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    put = lambda a, t=torch.int32: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    op = case["op"]
    if op == "layout":
        n = case["requests"]
        seq = np.exp(host.uniform(0, math.log(case["context"] + 1), n)).astype(np.int64) - 1
        q = _query_lens(case, host)
        width = -(-(case["context"] + _most_new(case)) // PAGE)
        used = -(-seq // PAGE)
        pages = host.permutation(int(used.sum()) + int((-(-(seq + q) // PAGE)).sum())).astype(np.int32)
        table = np.zeros((n, width), np.int32)
        table[np.arange(width)[None, :] < used[:, None]] = pages[: used.sum()]
        return dict(case=case, seq=put(seq), q=put(q), table=put(table), free=put(pages[used.sum():]),
                    prefix=put(np.array([case["prefix"]])))
    if op == "rope":
        x = normal(case["rows"], case["heads"], case["pitch"]).to(DTYPES[case["dtype"]])[..., case["pitch"] - case["width"]:]
        pos = put(host.integers(0, 163840, case["rows"]))
        return dict(case=case, x=x, pos=pos, inv=_inv_freq(case["rot"], case["base"], case["factor"]).cuda())
    if op == "append":
        n = case["rows"]
        kv = (normal(n, case["pitch"]) * 1.5).to(DTYPES[case["dtype"]])[:, case["pitch"] - DC - DP:]
        slots = host.permutation(case["pages"] * PAGE)[:n]
        slots[host.permutation(n)[: case["skip"]]] = -1
        return dict(case=case, kv=kv, w=(1 + 0.1 * normal(DC)).to(torch.bfloat16), slots=put(slots),
                    pos=put(host.integers(0, 163840, n)), inv=_inv_freq(DP, 10000.0, 40.0).cuda(),
                    ckv=(normal(case["pages"], PAGE, DC) * 0.5).to(torch.bfloat16),
                    kpe=(normal(case["pages"], PAGE, DP) * 0.5).to(torch.bfloat16))
    t, per, h = case["tokens"], case["per"], case["heads"]
    requests = t // per
    lens = host.integers(0, case["own"] + 1, requests)  # own rows of a request before this step's tokens
    token_lens = (lens[:, None] + 1 + np.arange(per)[None, :]).reshape(-1)
    own_pages = -(-(lens + per) // PAGE)
    first = -(-case["prefix"] // PAGE)
    pages = host.permutation(first + int(own_pages.sum())).astype(np.int32)
    table = np.zeros((requests, int(own_pages.max())), np.int32)
    table[np.arange(table.shape[1])[None, :] < own_pages[:, None]] = pages[first:]
    return dict(case=case, qn=normal(t, h, DC).to(torch.bfloat16), qp=normal(t, h, DP).to(torch.bfloat16),
                ckv=(normal(len(pages), PAGE, DC) * 0.5).to(torch.bfloat16),
                kpe=(normal(len(pages), PAGE, DP) * 0.5).to(torch.bfloat16),
                pages=put(pages[:first]), prefix=put(np.array([case["prefix"]])), table=put(table),
                lens=put(token_lens), request=put(np.repeat(np.arange(requests), per)))


# ------------------------------------------------------------ plain forms
def _plain_layout(s):
    rows, seq, q, free = s["case"]["rows"], s["seq"].long(), s["q"].long(), s["free"].long()
    table = s["table"]
    have, need = (seq + PAGE - 1) // PAGE, (seq + q + PAGE - 1) // PAGE
    taken = torch.cumsum(need - have, 0)
    start = taken - (need - have)
    col = torch.arange(table.shape[1], device=seq.device)
    new = (col >= have[:, None]) & (col < need[:, None])
    at = torch.where(new, start[:, None] + col - have[:, None], 0)
    # in place, as the table is the caller's; entries of other pages stay
    table.copy_(torch.where(new, free[at.clamp(max=max(0, free.numel() - 1))], table.long()))
    ends = torch.cumsum(q, 0)
    i = torch.arange(rows, device=seq.device)
    request = torch.searchsorted(ends, i, right=True)
    live = request < seq.numel()
    request = torch.where(live, request, 0)
    own_pos = i - (ends - q)[request] + seq[request]
    page = table.long()[request, torch.where(live, own_pos // PAGE, 0)]
    slot = torch.where(live, page * PAGE + own_pos % PAGE, -1)
    position = torch.where(live, own_pos + s["prefix"].long(), 0)
    visible = torch.where(live, own_pos + 1, 0)
    to = lambda v: v.to(torch.int32)  # noqa: E731
    return dict(table=table, slots=to(slot), positions=to(position), request=to(request), lens=to(visible),
                pages_used=to(taken[-1:]))


def _turned(x, pos, inv, layout, sign):
    """x [.., heads, rot] in 32 bits turned by position * inv, the angles in 64 bits."""
    angle = pos.double()[:, None, None] * inv
    c, s = torch.cos(angle).float(), torch.sin(angle).float() * sign
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _plain_rope(s):
    c, x = s["case"], s["x"]
    lo, hi = c["offset"], c["offset"] + c["rot"]
    turned = _turned(x[..., lo:hi].float(), s["pos"], s["inv"], c["layout"], -1.0 if c["inverse"] else 1.0)
    return torch.cat((x[..., :lo], turned.to(x.dtype), x[..., hi:]), -1)


def _plain_append(s):
    kv, slots = s["kv"].float(), s["slots"].long()
    latent = kv[:, :DC]
    latent = latent * torch.rsqrt((latent * latent).mean(-1, keepdim=True) + 1e-6) * s["w"].float()
    pe = _turned(kv[:, None, DC:], s["pos"], s["inv"], s["case"]["layout"], 1.0)[:, 0]
    keep = slots >= 0
    s["ckv"].view(-1, DC)[slots[keep]] = latent[keep].to(torch.bfloat16)
    s["kpe"].view(-1, DP)[slots[keep]] = pe[keep].to(torch.bfloat16)
    return dict(ckv=s["ckv"], kpe=s["kpe"])


def _plain_prefix(s):
    c = s["case"]
    t, h, lp = c["tokens"], c["heads"], c["prefix"]
    q = torch.cat((s["qn"], s["qp"]), -1).float()
    rows = torch.arange(lp, device=q.device)
    at = s["pages"].long()[rows // PAGE] * PAGE + rows % PAGE
    ckv, kpe = s["ckv"].view(-1, DC), s["kpe"].view(-1, DP)
    k = torch.cat((ckv[at], kpe[at]), -1).float()
    table = s["table"].long()
    cols = torch.arange(table.shape[1] * PAGE, device=q.device)
    at = (table[:, cols // PAGE] * PAGE + cols % PAGE)
    k_own = torch.cat((ckv[at], kpe[at]), -1).float()                        # [requests, own rows, 576]
    q_own = q.view(-1, c["per"] * h, DC + DP)                                 # the tokens of a request together
    s1 = (q.view(t * h, -1) @ k.T).view(t, h, lp) * SM_SCALE
    s2 = torch.bmm(q_own, k_own.transpose(1, 2)).view(t, h, -1) * SM_SCALE
    s2 = s2.masked_fill(cols >= s["lens"].long()[:, None, None], -math.inf)
    top = torch.maximum(s1.amax(-1), s2.amax(-1))
    p1, p2 = torch.exp(s1 - top[..., None]), torch.exp(s2 - top[..., None])
    total = p1.sum(-1) + p2.sum(-1)
    o = (p1.view(t * h, lp) @ k[:, :DC]).view(t, h, DC)
    o = o + torch.bmm(p2.view(-1, c["per"] * h, cols.numel()), k_own[..., :DC]).view(t, h, DC)
    return dict(out=(o / total[..., None]).to(torch.bfloat16), lse=(top + torch.log(total)) / math.log(2.0))


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"layout": _plain_layout, "rope": _plain_rope, "append": _plain_append, "prefix": _plain_prefix}[c["op"]](s)
    import flashinfer_repo_b200 as fi
    if c["op"] == "layout":
        r = fi.step_layout(s["seq"], s["q"], s["table"], s["free"], c["rows"], prefix_len=s["prefix"])
        return dict(table=s["table"], slots=r.slots, positions=r.positions, request=r.token_request, lens=r.token_lens,
                    pages_used=r.pages_used)
    if c["op"] == "rope":
        return fi.apply_rope(s["x"], s["pos"], s["inv"], layout=c["layout"], offset=c["offset"], inverse=c["inverse"])
    if c["op"] == "append":
        fi.latent_cache_append(s["kv"], s["w"], s["pos"], s["slots"], s["inv"], s["ckv"], s["kpe"], layout=c["layout"])
        return dict(ckv=s["ckv"], kpe=s["kpe"])
    out, lse = fi.shared_prefix_attention(s["qn"], s["qp"], s["ckv"], s["kpe"], s["pages"], s["prefix"], s["table"], s["lens"],
                                          SM_SCALE, token_request=s["request"])
    return dict(out=out, lse=lse)


# ------------------------------------------------------- work and 64 bits
def work(case):
    op = case["op"]
    if op == "layout":
        # the lengths of one seed: a pass reads both length vectors and the pages that it hands out and writes four words a row
        q = _query_lens(case, np.random.default_rng(0))
        pages = int((q // PAGE).sum()) + case["requests"] // PAGE
        return {"bytes": 8 * case["requests"] + 8 * pages + 4 * int((q > 0).sum()) + 16 * case["rows"], "flops": 0}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case.get("dtype", "bf16")]
    if op == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["width"] * size + 4 * case["rows"] + 4 * case["rot"], "flops": 3 * n * case["rot"]}
    if op == "append":
        n = case["rows"] - case["skip"]
        return {"bytes": n * (DC + DP) * (size + 2) + 8 * case["rows"] + 2 * DC, "flops": n * (4 * DC + 3 * DP)}
    t, h, requests = case["tokens"], case["heads"], case["tokens"] // case["per"]
    mean_own = case["own"] / 2  # lengths are uniform up to `own`
    rows = case["prefix"] + requests * (mean_own + case["per"])
    return {"bytes": rows * (DC + DP) * 2 + t * h * ((DC + DP) * 2 + DC * 2 + 4) + 4 * (rows / PAGE + 2 * t),
            "flops": 2 * t * h * (DC + DP + DC) * (case["prefix"] + mean_own + (case["per"] + 1) / 2)}


def _exact_turn(x, pos, inv, layout, inverse):
    """Rotation as a product of complex numbers."""
    x = x.double()
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous() if layout == "interleaved"
                              else x.unflatten(-1, (2, -1)).transpose(-1, -2).contiguous())
    angle = torch.outer(pos.double(), inv.double())[:, None, :]
    z = z * torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    z = torch.view_as_real(z)
    return z.flatten(-2) if layout == "interleaved" else z.transpose(-1, -2).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layout":
        seq, q, free = (s[k].tolist() for k in ("seq", "q", "free"))
        table = s["table"].cpu().numpy().copy()
        out = np.zeros((4, case["rows"]), np.int32)
        out[0] = -1
        row = used = 0
        for b in range(len(seq)):
            for i in range(q[b]):
                at = seq[b] + i
                if at % PAGE == 0:
                    table[b, at // PAGE] = free[used]
                    used += 1
                out[:, row] = table[b, at // PAGE] * PAGE + at % PAGE, case["prefix"] + at, b, at + 1
                row += 1
        return dict(table=table, slots=out[0], positions=out[1], request=out[2], lens=out[3], pages_used=np.array([used], np.int32))
    if case["op"] == "rope":
        y = s["x"].double().clone()
        part = slice(case["offset"], case["offset"] + case["rot"])
        y[..., part] = _exact_turn(y[..., part], s["pos"], s["inv"], case["layout"], case["inverse"])
        return y
    if case["op"] == "append":
        ckv, kpe, kv = s["ckv"].double(), s["kpe"].double(), s["kv"].double()
        norm = kv[:, :DC] / torch.sqrt(kv[:, :DC].pow(2).sum(-1, keepdim=True) / DC + 1e-6) * s["w"].double()
        pe = _exact_turn(kv[:, None, DC:], s["pos"], s["inv"], case["layout"], False)[:, 0]
        at = s["slots"].long()
        live = (at >= 0).nonzero()[:, 0]
        ckv[at[live] // PAGE, at[live] % PAGE] = norm[live]
        kpe[at[live] // PAGE, at[live] % PAGE] = pe[live]
        return dict(ckv=ckv, kpe=kpe)
    # one token after the other, all that it sees in one list of rows
    lens, request, table = s["lens"].tolist(), s["request"].tolist(), s["table"].long()
    prefix = (s["pages"].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()[: case["prefix"]]
    ckv, kpe = s["ckv"].view(-1, DC), s["kpe"].view(-1, DP)
    pre_c, pre_p = ckv[prefix].double(), kpe[prefix].double()
    out, lse = [], []
    for t in range(case["tokens"]):
        at = (table[request[t]][:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()[: lens[t]]
        c, p = torch.cat((pre_c, ckv[at].double())), torch.cat((pre_p, kpe[at].double()))
        z = (s["qn"][t].double() @ c.T + s["qp"][t].double() @ p.T) * SM_SCALE
        each = torch.logsumexp(z, -1)
        out.append(torch.exp(z - each[:, None]) @ c)
        lse.append(each / math.log(2.0))
    return dict(out=torch.stack(out), lse=torch.stack(lse))
