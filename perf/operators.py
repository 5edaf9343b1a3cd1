"""Measured cases of the token-mixing operators: the gated delta rule (prompt and single-token forms) and
attention over a paged INT8 cache (append, read back, attend).

Sizes: the gated delta rule's head layout is the one behind this package's grouped projection of 12288 rows
(8192 of q, k and v: 16 key heads and 32 value heads of 128; 4096 of the z branch).  Attention uses 16 query
heads over 4 cached heads of 256.  Drawn cases vary heads, widths, page sizes and lengths around these.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
CHUNK = 64                # rows a chunk of the plain gated delta rule


# ------------------------------------------------------------------------------------------------------- cases
def listed():
    gdn = dict(k_heads=16, v_heads=32, dk=128, dv=128, normalize=True)
    att = dict(kv_heads=4, group=4, dim=256, page=64)
    return [
        # one short request entering the model: latency of the chunked form
        dict(name="gdn prompt 1x96", op="gdn_prefill", batch=1, tokens=96, carry=False, **gdn),
        # a packed batch of ragged requests that continue from kept states (chunked prefill)
        dict(name="gdn prompts 8, 4001 rows", op="gdn_prefill", batch=8, tokens=4001, carry=True, **gdn),
        # one long prompt: nothing but heads to run in parallel
        dict(name="gdn prompt 1x8192", op="gdn_prefill", batch=1, tokens=8192, carry=False, **gdn),
        # a full prompt batch: throughput
        dict(name="gdn prompts 16, 32768 rows", op="gdn_prefill", batch=16, tokens=32768, carry=False, **gdn),
        # single-token steps: one stream, an odd batch, a full server
        dict(name="gdn step 1", op="gdn_decode", batch=1, **gdn),
        dict(name="gdn step 37", op="gdn_decode", batch=37, **gdn),
        dict(name="gdn step 512", op="gdn_decode", batch=512, **gdn),
        # one new row for each of 64 sequences, then the touched pages read back
        dict(name="append 64x1", op="append", batch=64, rows=64, cached=64 * 1000 + 13, kv_heads=4, dim=256, page=64),
        # ragged prompts entering the cache, then read back
        dict(name="append 8, 8191 rows", op="append", batch=8, rows=8191, cached=1001, kv_heads=4, dim=256, page=64),
        # one stream's step over a mid-sized context: latency, work split over the context
        dict(name="attend 1x4097", op="attend", batch=1, rows=1, cached=4097, **att),
        # a full server's step
        dict(name="attend 64, 261000 cached", op="attend", batch=64, rows=64, cached=261000, **att),
        # a chunk of four prompts over what is already cached
        dict(name="attend 4, 2048 rows", op="attend", batch=4, rows=2048, cached=16000, **att),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gdn_prefill", "gdn_decode", "append", "attend_step", "attend_rows"])
    if op.startswith("gdn"):
        k_heads = rng.choice([2, 4, 8, 16])
        case = dict(op=op, k_heads=k_heads, v_heads=k_heads * rng.choice([1, 2]), dk=rng.choice([64, 128, 128]),
                    dv=rng.choice([64, 128, 128]), normalize=rng.random() < 0.75)
        if op == "gdn_decode":
            return dict(case, batch=_log(rng, 1, 512))
        tokens = _log(rng, 1, 32768)
        return dict(case, tokens=tokens, batch=min(tokens, _log(rng, 1, 32)), carry=rng.random() < 0.5)
    dim = rng.choice([64, 128, 256])
    case = dict(kv_heads=rng.choice([1, 2, 4] if dim == 256 else [1, 2, 4, 8]), dim=dim, page=rng.choice([16, 32, 64]))
    if op == "append":
        rows = _log(rng, 1, 8191)
        batch = min(rows, _log(rng, 1, 64))
        return dict(case, op=op, batch=batch, rows=rows, cached=_log(rng, 1, 65536))
    case["group"] = rng.choice([x for x in (1, 2, 4, 8) if x * case["kv_heads"] <= 16])
    if op == "attend_step":
        batch = _log(rng, 1, 128)
        return dict(case, op="attend", batch=batch, rows=batch, cached=batch * _log(rng, 1, 261000 // batch))
    rows = _log(rng, 2, 2048)
    batch = min(rows, _log(rng, 1, 8))
    return dict(case, op="attend", batch=batch, rows=rows, cached=rows + _log(rng, 1, 14000))


def _split(total, parts, least=0):
    """`total` as `parts` ragged whole numbers of at least `least`: the same for a case whatever the seed."""
    rng = random.Random(total * 7919 + parts)
    weights = [rng.uniform(0.25, 1.75) for _ in range(parts)]
    free, whole = total - least * parts, sum(weights)
    ends, acc = [], 0.0
    for w in weights:
        acc += w
        ends.append(int(free * acc / whole + 0.5))
    ends[-1] = free
    return [least + e - s for s, e in zip([0] + ends[:-1], ends)]


def _lengths(case):
    """(new rows, rows cached before them) of each sequence."""
    rows = _split(case["rows"], case["batch"], 1)
    if case["op"] == "append":
        return rows, _split(case["cached"], case["batch"])
    # `cached` counts the rows under attention, the newest ones among them
    older = _split(max(0, case["cached"] - case["rows"]), case["batch"])
    return rows, older


# ----------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed) % (1 << 62))
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = dict(case=case)
    if case["op"].startswith("gdn"):
        n = case["tokens"] if case["op"] == "gdn_prefill" else case["batch"]
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["dk"], case["dv"]
        size = 1.0 if case["normalize"] else dk ** -0.5
        # keys and queries share a direction per head, as trained ones do; q, k and v are slices of one
        # projection's rows
        qkv = normal(n, hk * dk * 2 + hv * dv)
        qkv[:, :hk * dk * 2] += 0.5 * normal(1, hk * dk).repeat(1, 2)
        qkv[:, :hk * dk * 2] *= size
        qkv = qkv.to(torch.bfloat16)
        s["q"] = qkv[:, :hk * dk].view(n, hk, dk)
        s["k"] = qkv[:, hk * dk:2 * hk * dk].view(n, hk, dk)
        s["v"] = qkv[:, 2 * hk * dk:].view(n, hv, dv)
        rate = 1.0 + 15.0 * uniform(1, hv)
        s["g"] = -rate * torch.exp(math.log(1e-3) + uniform(n, hv) * math.log(100.0))      # log of the decay
        s["beta"] = torch.sigmoid(normal(n, hv))
        slots = case["batch"] + 3
        s["state"] = normal(slots, hv, dk, dv) * 0.1
        s["slots"] = torch.randperm(slots, generator=g, device=DEVICE)[:case["batch"]].to(torch.int32)
        if case["op"] == "gdn_prefill":
            s["lens"] = _split(n, case["batch"], 1)
            s["cu"] = _offsets(s["lens"])
        return s
    rows, older = _lengths(case)
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    n, per = sum(rows), [-(-(a + b) // page) for a, b in zip(rows, older)]
    pages = sum(per) + 5
    ids = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    s["tables"] = torch.zeros(case["batch"], max(per), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, m in enumerate(per):
        s["tables"][b, :m] = ids[at:at + m]
        at += m
    s["rows"], s["older"] = rows, older
    s["cu"] = _offsets(rows)
    for x in ("k", "v"):
        codes = torch.randint(-127, 128, (pages, heads, page, dim), generator=g, device=DEVICE, dtype=torch.int8)
        s[x + "8"] = codes
        s[x + "_scale"] = (1.0 + 3.0 * uniform(pages, heads)) / 127.0
    if case["op"] == "append":
        for x in ("k", "v"):
            s[x] = (normal(n, heads, dim) * torch.exp(0.5 * normal(n, heads, 1))).to(torch.bfloat16)
        s["lengths"] = torch.tensor(older, dtype=torch.int32, device=DEVICE)
        s["first"] = [o // page * page for o in older]                    # read back from the first touched page on
        s["starts"] = torch.tensor(s["first"], dtype=torch.int32, device=DEVICE)
        s["back"] = _offsets([o + r - f for o, r, f in zip(older, rows, s["first"])])
        s["back_rows"] = int(sum(older) + n - sum(s["first"]))
    else:
        s["q"] = normal(n, heads * case["group"], dim).to(torch.bfloat16)
        s["lengths"] = torch.tensor([a + b for a, b in zip(rows, older)], dtype=torch.int32, device=DEVICE)
    return s


def _offsets(lens):
    at = [0]
    for x in lens:
        at.append(at[-1] + x)
    return torch.tensor(at, dtype=torch.int32, device=DEVICE)


# -------------------------------------------------------------------------------------------------------- runs
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_prefill(s):
    from reax_engine_runtime_v3_b200 import gated_delta
    c = s["case"]
    out = gated_delta.prefill(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], cu_seqlens=s["cu"],
                              slots=s["slots"], carry=c["carry"], normalize=c["normalize"])
    return dict(out=out, state=s["state"])


def _own_decode(s):
    from reax_engine_runtime_v3_b200 import gated_delta
    out = gated_delta.decode(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], slots=s["slots"],
                             normalize=s["case"]["normalize"])
    return dict(out=out, state=s["state"])


def _own_append(s):
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    cache = Int8Cache(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    cache.append(s["k"], s["v"], s["tables"], s["lengths"], cu_seqlens=s["cu"])
    k, v = cache.read(s["tables"], s["starts"], s["back"], s["back_rows"])
    return dict(k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_attend(s):
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    cache = Int8Cache(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    out, lse = cache.attend(s["q"], s["tables"], s["lengths"], cu_seqlens=s["cu"], max_rows=max(s["rows"]),
                            return_lse=True)
    return dict(out=out, lse=lse)


_own = dict(gdn_prefill=_own_prefill, gdn_decode=_own_decode, append=_own_append, attend=_own_attend)


def _qk(s):
    """q (scaled) and k for every value head in float32 [rows, v_heads, dk]."""
    c = s["case"]
    q, k = s["q"].float(), s["k"].float()
    if c["normalize"]:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    each = c["v_heads"] // c["k_heads"]
    return (q * c["dk"] ** -0.5).repeat_interleave(each, 1), k.repeat_interleave(each, 1)


def _plain_decode(s):
    q, k = _qk(s)
    slots = s["slots"].long()
    state = s["state"][slots] * torch.exp(s["g"])[..., None, None]
    u = (s["v"].float() - (k[..., None] * state).sum(2)) * s["beta"][..., None]
    state = state + k[..., None] * u[..., None, :]
    s["state"][slots] = state
    return dict(out=(q[..., None] * state).sum(2).to(torch.bfloat16), state=s["state"])


def _plain_prefill(s):
    """Chunks of CHUNK rows.  Within a chunk, with G the running sum of g, the rows' corrections solve
    (I + A) V' = beta (V - e^G K S), A = tril(beta_i e^(G_i - G_j) k_i.k_j, -1); the chunks' states follow
    S <- M S + B one after the other, and all else is batched."""
    c, lens = s["case"], s["lens"]
    q, k = _qk(s)
    n, hv, dk = k.shape
    dv = c["dv"]
    # chunks ordered by their place in the sequence, longest sequence first, so that those at one place lie together
    order = sorted(range(len(lens)), key=lambda b: -lens[b])
    begin = [0]
    for x in lens:
        begin.append(begin[-1] + x)
    most = -(-max(lens) // CHUNK)
    places = [[b for b in order if lens[b] > at * CHUNK] for at in range(most)]
    first = torch.tensor([begin[b] + at * CHUNK for at in range(most) for b in places[at]], device=DEVICE)
    count = torch.tensor([min(CHUNK, lens[b] - at * CHUNK) for at in range(most) for b in places[at]], device=DEVICE)
    row = torch.arange(CHUNK, device=DEVICE)
    real = row[None] < count[:, None]                                                   # [chunks, CHUNK]
    index = torch.where(real, first[:, None] + row[None], 0)
    pick = lambda x: (x[index] * real.view(*real.shape, *[1] * (x.dim() - 1))).transpose(1, 2)  # noqa: E731
    q, k, v = pick(q), pick(k), pick(s["v"].float())                                    # [chunks, heads, CHUNK, d]
    g, beta = pick(s["g"]).cumsum(-1), pick(s["beta"])[..., None]
    below = row[:, None] >= row[None]
    decay = torch.exp(torch.where(below, g[..., :, None] - g[..., None, :], float("-inf")))
    a = (beta * decay * (k @ k.transpose(-1, -2))).tril(-1)
    t = torch.eye(CHUNK, device=DEVICE).expand_as(a).clone()                            # (I + a)^-1, block by block
    for h in (1, 2, 4, 8, 16, 32):
        m = CHUNK // (2 * h)
        tb = t.view(-1, m, 2 * h, m, 2 * h).diagonal(dim1=1, dim2=3).permute(0, 3, 1, 2)
        ab = a.reshape(-1, m, 2 * h, m, 2 * h).diagonal(dim1=1, dim2=3).permute(0, 3, 1, 2)
        tb[..., h:, :h] = -(tb[..., h:, h:] @ ab[..., h:, :h] @ tb[..., :h, :h])
    eg, last = torch.exp(g)[..., None], g[..., -1:]
    w, u = t @ (beta * eg * k), t @ (beta * v)
    late = (torch.exp(last - g)[..., None] * k).transpose(-1, -2)
    mm = torch.exp(last)[..., None] * torch.eye(dk, device=DEVICE) - late @ w
    bb = late @ u
    slots = s["slots"].long()[torch.tensor(order, device=DEVICE)]
    state = s["state"][slots] if c["carry"] else torch.zeros(len(lens), hv, dk, dv, device=DEVICE)
    held = torch.empty(len(first), hv, dk, dv, device=DEVICE)                           # the state before each chunk
    at = 0
    for p in places:                                                                    # in sequence by definition
        m = len(p)
        held[at:at + m] = state[:m]
        state[:m] = bb[at:at + m] + mm[at:at + m] @ state[:m]
        at += m
    s["state"][slots] = state
    o = eg * q @ held + (decay * (q @ k.transpose(-1, -2))) @ (u - w @ held)
    out = torch.empty(n, hv, dv, dtype=torch.bfloat16, device=DEVICE)
    out[index[real]] = o.transpose(1, 2)[real].to(torch.bfloat16)
    return dict(out=out, state=s["state"])


def _plain_append(s):
    """Each page and head keeps one scale, the largest |x| / 127 so far; where it grows, the page's older codes
    are rounded anew."""
    page = s["case"]["page"]
    older, rows = s["lengths"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    n = s["k"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(older), device=DEVICE), rows, output_size=n)
    at = older[seq] + torch.arange(n, device=DEVICE) - s["cu"][:-1].long()[seq]
    where = s["tables"][seq, at // page].long()
    back = torch.repeat_interleave(torch.arange(len(older), device=DEVICE), (s["back"][1:] - s["back"][:-1]).long(),
                                   output_size=s["back_rows"])
    place = s["starts"].long()[back] + torch.arange(s["back_rows"], device=DEVICE) - s["back"][:-1].long()[back]
    from_page = s["tables"][back, place // page].long()
    got = dict(k_scale=s["k_scale"], v_scale=s["v_scale"])
    touched = older // page
    kept = older % page                                                                 # rows of a page begun before
    begun = kept > 0
    old_page = s["tables"][torch.arange(len(older), device=DEVICE), torch.where(begun, touched, 0)].long()
    for x in ("k", "v"):
        new, codes, scale = s[x].float(), s[x + "8"], s[x + "_scale"]
        new_scale = torch.zeros_like(scale)
        new_scale[where] = 1e-12 / 127.0
        need = new.abs().amax(-1).clamp(min=1e-12) / 127.0                              # [rows, heads]
        new_scale.scatter_reduce_(0, where[:, None].expand_as(need), need, "amax")
        was = torch.where(begun[:, None], scale[old_page], 0.0)                         # [sequences, heads]
        now = torch.where(begun[:, None], torch.maximum(new_scale[old_page], was), 0.0)
        again = torch.round(codes[old_page].float() * torch.where(now > was, was / now, 1.0)[..., None, None])
        held = torch.arange(page, device=DEVICE)[None] < kept[:, None]
        now_codes = torch.where(held[:, None, :, None], again.to(torch.int8), codes[old_page])
        codes[old_page[begun]] = now_codes[begun]
        new_scale[old_page[begun]] = now[begun]
        hit = new_scale > 0
        scale.copy_(torch.where(hit, new_scale, scale))
        codes[where, :, at % page] = torch.round(new / scale[where][..., None]).clamp(-127, 127).to(torch.int8)
        got[x] = (codes[from_page, :, place % page].float() * scale[from_page][..., None]).to(torch.bfloat16)
    return got


def _plain_attend(s):
    c = s["case"]
    page, heads, group, dim = c["page"], c["kv_heads"], c["group"], c["dim"]
    batch, most, n = c["batch"], max(s["rows"]), s["q"].shape[0]
    rows, lengths = (s["cu"][1:] - s["cu"][:-1]).long(), s["lengths"].long()
    seq = torch.repeat_interleave(torch.arange(batch, device=DEVICE), rows, output_size=n)
    place = torch.arange(n, device=DEVICE) - s["cu"][:-1].long()[seq]
    q = torch.zeros(batch, most, heads, group, dim, device=DEVICE)
    q[seq, place] = s["q"].float().view(n, heads, group, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim) * dim ** -0.5
    pages = s["tables"].long()
    spread = lambda x: x.permute(0, 2, 1, 3, 4).reshape(batch, heads, -1, dim)  # noqa: E731
    k = spread(s["k8"][pages].float() * s["k_scale"][pages][..., None, None])
    score = (q @ k.transpose(-1, -2)).view(batch, heads, group, most, -1)
    del k
    limit = lengths[:, None] - rows[:, None] + torch.arange(most, device=DEVICE)[None]  # the last place a row sees
    seen = torch.arange(score.shape[-1], device=DEVICE)[None, None] <= limit[..., None]
    score = torch.where(seen[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    del score
    total = p.sum(-1, keepdim=True)
    v = spread(s["v8"][pages].float() * s["v_scale"][pages][..., None, None])
    out = (p.view(batch, heads, group * most, -1) @ v).view(batch, heads, group, most, dim) / total
    lse = (top + torch.log(total))[..., 0]
    flat = lambda x: x[seq, :, :, place].reshape(n, heads * group, *x.shape[4:])  # noqa: E731
    return dict(out=flat(out).to(torch.bfloat16), lse=flat(lse))


_plain = dict(gdn_prefill=_plain_prefill, gdn_decode=_plain_decode, append=_plain_append, attend=_plain_attend)


# -------------------------------------------------------------------------------------------------------- work
def work(case):
    b = case["batch"]
    if case["op"].startswith("gdn"):
        n = case.get("tokens", b)
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["dk"], case["dv"]
        reads = 2 if case["op"] == "gdn_decode" or case["carry"] else 1
        # rows in and out, and the states; three products of a dk x dv matrix with a vector for each row and head
        return {"bytes": n * (2 * hk * dk * 2 + 2 * hv * dv * 2 + 8 * hv) + reads * b * hv * dk * dv * 4,
                "flops": n * hv * 6 * dk * dv}
    rows, older = _lengths(case)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    scales = 8 * heads * sum(-(-(r + o) // page) for r, o in zip(rows, older))
    if case["op"] == "append":
        back = sum(r + o % page for r, o in zip(rows, older))
        # rows in, codes out; then codes in, rows out
        return {"bytes": 2 * heads * dim * (3 * sum(rows) + 3 * back), "flops": 2 * heads * dim * 2 * (sum(rows) + back)}
    pairs = sum(r * o + r * (r + 1) // 2 for r, o in zip(rows, older))
    heads_q = heads * case["group"]
    return {"bytes": 2 * heads * dim * sum(r + o for r, o in zip(rows, older)) + scales
            + sum(rows) * heads_q * (4 * dim + 4), "flops": 4 * heads_q * dim * pairs}


# ------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions, in 64 bits: the gated delta rule row by row, softmax attention sequence by sequence."""
    s = prepare(case, seed)
    if case["op"] == "append":
        scales = {x: _exact_scales(s, x) for x in ("k", "v")}
        return dict(k=None, v=None, k_scale=scales["k"], v_scale=scales["v"])
    if case["op"] == "attend":
        return _exact_attend(s)
    lens = s.get("lens") or [1] * case["batch"]
    hv, dk = case["v_heads"], case["dk"]
    each = hv // case["k_heads"]
    slots = s["slots"].long()
    final = s["state"].double()
    state = final[slots] if case.get("carry", True) else torch.zeros_like(final[slots])
    out = torch.empty(*s["v"].shape, dtype=torch.float64, device=DEVICE)
    begin = torch.tensor([sum(lens[:b]) for b in range(len(lens))], device=DEVICE)
    long = torch.tensor(lens, device=DEVICE)
    order = torch.argsort(long, descending=True)
    active = [sum(x > t for x in lens) for t in range(max(lens))]
    q, k, v = (s[x].double() for x in "qkv")
    if case["normalize"]:
        q, k = (x / torch.sqrt(torch.sum(x * x, -1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = q.repeat_interleave(each, 1) / math.sqrt(dk), k.repeat_interleave(each, 1)
    alpha, beta = torch.exp(s["g"].double()), s["beta"].double()
    state, begin = state[order], begin[order]
    for t, m in enumerate(active):
        r = begin[:m] + t
        x = state[:m]
        x.mul_(alpha[r][..., None, None])
        old = torch.einsum("bhk,bhkv->bhv", k[r], x)
        x.add_(torch.einsum("bhk,bhv->bhkv", k[r], beta[r][..., None] * (v[r] - old)))
        out[r] = torch.einsum("bhk,bhkv->bhv", q[r], x)
    final[slots[order]] = state
    return dict(out=out, state=final)


def _exact_scales(s, x):
    page = s["case"]["page"]
    scale = s[x + "_scale"].double().clone()
    rows, cu, tables = s[x].double(), s["cu"].tolist(), s["tables"].tolist()
    for b, (n, older) in enumerate(zip(s["rows"], s["older"])):
        at = older
        while at < older + n:
            end = min(older + n, (at // page + 1) * page)
            most = rows[cu[b] + at - older:cu[b] + end - older].abs().amax((0, 2)) / 127
            where = tables[b][at // page]
            scale[where] = torch.maximum(scale[where], most) if at % page else most
            at = end
    return scale


def _exact_attend(s):
    c = s["case"]
    outs, lses, at = [], [], 0
    for b, (n, older) in enumerate(zip(s["rows"], s["older"])):
        length = n + older
        pages = s["tables"][b, :-(-length // c["page"])].long()
        seen = torch.arange(length, device=DEVICE)[None] <= older + torch.arange(n, device=DEVICE)[:, None]
        out = torch.empty(n, c["kv_heads"] * c["group"], c["dim"], dtype=torch.float64, device=DEVICE)
        lse = torch.empty(n, c["kv_heads"] * c["group"], dtype=torch.float64, device=DEVICE)
        for h in range(c["kv_heads"]):
            k, v = (torch.flatten(s[x + "8"][pages, h].double() * s[x + "_scale"][pages, h].double()[:, None, None],
                                  0, 1)[:length] for x in "kv")
            for i in range(h * c["group"], (h + 1) * c["group"]):
                score = (s["q"][at:at + n, i].double() @ k.T / math.sqrt(c["dim"])).masked_fill(~seen, -math.inf)
                lse[:, i] = torch.logsumexp(score, -1)
                out[:, i] = torch.exp(score - lse[:, i, None]) @ v
        outs.append(out)
        lses.append(lse)
        at += n
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
