"""Long-context serving over a paged cache, as cases that can be timed and compared: new rows rotated into the cache, the blocks that a query
reads chosen by a score over the blocks' bounds, and attention over those blocks.

A cache layer is [pages, 2, page, kv heads, dim].  Pages are cut into blocks; a complete block has, per kv head and channel, the largest and the
smallest of its keys as a whole number of steps, -127 to 127, rounded outward; a step is a power of two (`steps`).  Rows carry their request (`q_req`) and the number of
tokens they see (`q_kvlen`); `indptr` / `indices` hold the requests' pages.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
FIRST, LAST = 1, 2          # blocks that every row reads: the first of the sequence, the newest two
SEGMENT = 32                # neighbouring cached tokens that are about the same thing
LOWEST = 2.0 ** -100        # the smallest unit of a bound


def listed():
    return [
        # one stream being spoken, a frame's new token (16 query heads on 8, head dim 128)
        dict(name="append_decode_1", kind="append", rows=1, reqs=1, ctx=2000, heads=16, kv_heads=8, dim=128, rot=128, pairs="halves", page=128, block=64, dtype="bf16"),
        # continuous batching, neighbouring pairs over half of the head
        dict(name="append_decode_48", kind="append", rows=48, reqs=48, ctx=4000, heads=32, kv_heads=2, dim=128, rot=64, pairs="neighbours", page=128, block=64, dtype="bf16"),
        # three prompts of uneven length together, head dim 64 in fp16
        dict(name="append_prompt_2000_f16", kind="append", rows=2000, reqs=3, ctx=2500, heads=32, kv_heads=8, dim=64, rot=64, pairs="halves", page=16, block=16, dtype="f16"),
        # chunks of eight long prompts
        dict(name="append_prompt_16384", kind="append", rows=16384, reqs=8, ctx=8192, heads=32, kv_heads=8, dim=128, rot=128, pairs="halves", page=128, block=64, dtype="bf16"),
        # one request deep in a long session: 2048 blocks to choose from
        dict(name="select_decode_1", kind="select", rows=1, reqs=1, ctx=131072, heads=32, kv_heads=2, dim=128, page=128, block=64, top=32, dtype="bf16"),
        # 32 requests of a few thousand to 16 thousand tokens
        dict(name="select_decode_32", kind="select", rows=32, reqs=32, ctx=16384, heads=16, kv_heads=8, dim=128, page=128, block=32, top=48, dtype="bf16"),
        # two prompts' chunks behind long contexts, an odd number of rows
        dict(name="select_prompt_1001", kind="select", rows=1001, reqs=2, ctx=16000, heads=12, kv_heads=4, dim=128, page=128, block=64, top=32, dtype="bf16"),
        # a large chunk of one long prompt
        dict(name="select_prompt_4096", kind="select", rows=4096, reqs=1, ctx=32768, heads=16, kv_heads=8, dim=128, page=128, block=64, top=32, dtype="bf16"),
        # one stream: 512 tokens of its context
        dict(name="attend_decode_1", kind="attend", rows=1, reqs=1, ctx=2000, heads=16, kv_heads=8, dim=128, page=128, block=32, top=16, dtype="bf16"),
        # 64 requests, 2048 tokens each, head dim 64 in fp16
        dict(name="attend_decode_64_f16", kind="attend", rows=64, reqs=64, ctx=20000, heads=32, kv_heads=8, dim=64, page=64, block=32, top=64, dtype="f16"),
        # few requests with much to read: 16 query heads on a kv head, 8192 tokens each
        dict(name="attend_decode_4_long", kind="attend", rows=4, reqs=4, ctx=131072, heads=32, kv_heads=2, dim=128, page=128, block=128, top=64, dtype="bf16"),
        # a chunk of a long prompt, every row with its own blocks
        dict(name="attend_prompt_1024", kind="attend", rows=1024, reqs=1, ctx=16384, heads=16, kv_heads=8, dim=128, page=128, block=64, top=32, dtype="bf16"),
    ]


def cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    while True:
        kind = rng.choice(["append", "select", "attend"])
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 2, 128), (12, 4, 128), (32, 8, 128), (32, 8, 64), (14, 2, 64), (8, 8, 64), (32, 32, 128)])
        block = rng.choice([16, 32, 64, 128])
        case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, block=block, page=block * rng.choice([1, 1, 2, 3, 4]), dtype=rng.choice(["bf16", "bf16", "f16"]))
        prompt = rng.random() < 0.5
        if kind == "append":
            case["rot"] = rng.choice([dim, dim, dim // 2])
            case["pairs"] = rng.choice(["halves", "neighbours"])
            case["rows"] = log(17, 16384) if prompt else log(1, 128)
            case["reqs"] = rng.randint(1, min(8, case["rows"])) if prompt else case["rows"]
            case["ctx"] = max(log(64, 8192), -(-case["rows"] // case["reqs"]) * 2) if prompt else log(64, 16384)
        else:
            case["top"] = log(FIRST + LAST + 1, 64)
            case["rows"] = log(17, 4096) if prompt else log(1, 64)
            case["reqs"] = rng.randint(1, 4) if prompt else case["rows"]
            case["ctx"] = max(log(256, 131072), -(-case["rows"] // case["reqs"]) * 2)
        cache = case["reqs"] * case["ctx"] * kv_heads * dim * 4
        gathered = case["rows"] * kv_heads * case.get("top", 0) * block * dim if kind == "attend" else 0
        scores = case["rows"] * kv_heads * case["reqs"] * (case["ctx"] // block) if kind == "select" else 0
        if kind == "select" and 0.6 * case["ctx"] // block <= case["top"] + 1:
            continue                      # nothing to choose
        roof = max(cost(c) for c in listed() if c["kind"] == kind)
        if cache <= 2 ** 32 and gathered <= 2 ** 31 and scores <= 2 ** 27 and cost(case) <= roof:
            return case


def make_plan(case, gen):
    """Lengths, pages and rows of the requests, on the host: the first request is as long as the case says, the others 60 to 100 % of it.
    The lengths are the case's own, the pages' order the seed's."""
    reqs, rows, ctx, page = case["reqs"], case["rows"], case["ctx"], case["page"]
    by_case = torch.Generator().manual_seed(rows + ctx)
    share = 0.6 + 0.4 * torch.rand(reqs, generator=by_case, dtype=torch.float64)
    share[0] = 1.0
    new = torch.full((reqs,), rows // reqs)
    new[: rows % reqs] += 1
    if reqs > 1 and rows > 4 * reqs:      # uneven chunks of the same sum
        shift = (new[0] * torch.rand(reqs // 2, generator=by_case, dtype=torch.float64) * 0.7).long()
        new[: reqs // 2] -= shift
        new[reqs - reqs // 2:] += shift
    kvlen = torch.maximum((ctx * share).long(), new)
    n_pages = (kvlen + page - 1) // page
    indptr = torch.cat([torch.zeros(1, dtype=torch.long), n_pages.cumsum(0)])
    total = int(indptr[-1]) + 1           # one page is nobody's
    indices = torch.randperm(total, generator=gen)[: total - 1]
    q_req = torch.repeat_interleave(torch.arange(reqs), new)
    at = torch.arange(rows) - torch.repeat_interleave(new.cumsum(0) - new, new)
    q_kvlen = (kvlen - new)[q_req] + at + 1
    pos = q_kvlen - 1
    pages = indices[indptr[q_req] + pos // page]

    def up(t):
        return t.to(device=DEV, dtype=torch.int32)
    return dict(q_req=up(q_req), q_kvlen=up(q_kvlen), indptr=up(indptr), indices=up(indices), pos=up(pos), pages=up(pages), slots=up(pos % page),
                n_pages=total, max_kvlen=int(kvlen.max()))


def make_bounds(kv, block):
    """Bounds of every block of a cache layer, [pages, kv heads, blocks, 2, dim] (largest, smallest), and their units."""
    p, _, page, h, d = kv.shape
    k = kv[:, 0].float().reshape(p, page // block, block, h, d)
    most, least = k.amax(2), k.amin(2)
    amax = torch.maximum(most.abs(), least.abs()).amax(-1)
    step = torch.ldexp(torch.ones_like(amax), torch.frexp(amax)[1] - 7)
    step = torch.where(amax > 127 * step, 2 * step, step).clamp(min=LOWEST)
    hi, lo = torch.ceil(most / step[..., None]), torch.floor(least / step[..., None])
    return torch.stack([hi, lo], dim=3).to(torch.int8).transpose(1, 2).contiguous(), step.transpose(1, 2).contiguous()


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device=DEV).manual_seed(seed)
    dtype, rows, page, h, d = DTYPES[case["dtype"]], case["rows"], case["page"], case["kv_heads"], case["dim"]
    group = case["heads"] // h
    s = make_plan(case, host)

    def normal(*shape):
        return torch.randn(*shape, generator=dev, device=DEV)
    # what tokens are about: neighbours share a topic, a query looks for one; channels have their own mean, as keys of real layers do
    topics, mean = 0.6 * normal(64, h, d), 0.5 * normal(h, d)
    parts = -(-page // SEGMENT)
    about = torch.randint(64, (s["n_pages"], parts), generator=dev, device=DEV).repeat_interleave(SEGMENT, 1)[:, :page]
    kv = torch.empty(s["n_pages"], 2, page, h, d, dtype=dtype, device=DEV)
    kv[:, 0] = (normal(s["n_pages"], page, h, d) + topics[about] + mean).to(dtype)
    kv[:, 1] = normal(s["n_pages"], page, h, d).to(dtype)
    wanted = topics[torch.randint(64, (rows // 16 + 1,), generator=dev, device=DEV).repeat_interleave(16)[:rows]]
    q = (normal(rows, h, group, d) + wanted[:, :, None]).reshape(rows, case["heads"] * d)
    s.update(case=case, kv=kv, scale=d ** -0.5)
    s["bounds"], s["steps"] = make_bounds(kv, case["block"])
    if case["kind"] == "append":
        # the projection's output holds q, k and v side by side
        kv_new = torch.cat([(normal(rows, h, d) + mean).reshape(rows, h * d), normal(rows, h * d)], 1)
        s["qkv"] = torch.cat([q, kv_new], 1).to(dtype)
        half = case["rot"] // 2
        angle = torch.arange(s["max_kvlen"], dtype=torch.float64, device=DEV)[:, None] * 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    else:
        s["q"] = q.reshape(rows, case["heads"], d).to(dtype)
    if case["kind"] == "attend":
        s["blocks"] = plain_select(s)
    return s


def split_qkv(s):
    c, qkv = s["case"], s["qkv"]
    at = [0, c["heads"] * c["dim"], (c["heads"] + c["kv_heads"]) * c["dim"], (c["heads"] + 2 * c["kv_heads"]) * c["dim"]]
    return [qkv[:, a:b].unflatten(1, (-1, c["dim"])) for a, b in zip(at, at[1:])]


def turn(x, cs, pairs):
    """The first 2 * cs.shape[1] channels turned by the row's angles: x cos is rounded, the other product is fused into the sum."""
    rot = 2 * cs.shape[1]
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    x = x.float()
    head, rest = x[..., :rot], x[..., rot:]
    a, b = (head[..., 0::2], head[..., 1::2]) if pairs == "neighbours" else (head[..., :rot // 2], head[..., rot // 2:])
    u = ((a * c).double() - b.double() * sn.double()).float()
    v = ((b * c).double() + a.double() * sn.double()).float()
    turned = torch.stack([u, v], -1).flatten(-2) if pairs == "neighbours" else torch.cat([u, v], -1)
    return torch.cat([turned, rest], -1)


def plain_append(s):
    c, kv = s["case"], s["kv"]
    q, k, v = split_qkv(s)
    cs = s["cos_sin"][s["pos"].long()]
    q_out = turn(q, cs, c["pairs"]).to(kv.dtype)
    page, slot = s["pages"].long(), s["slots"].long()
    kv[page, 0, slot] = turn(k, cs, c["pairs"]).to(kv.dtype)
    kv[page, 1, slot] = v
    # the blocks whose last token came with these rows
    done = (slot + 1) % c["block"] == 0
    page, part = page[done], slot[done] // c["block"]
    blocks = kv[:, 0].unflatten(1, (-1, c["block"]))[page, part]
    bounds, steps = make_bounds(blocks[:, None], c["block"])
    s["bounds"][page, :, part] = bounds[:, :, 0]
    s["steps"][page, :, part] = steps[:, :, 0]
    return q_out


def in_steps(q, kv_heads):
    """Query heads in 8-bit units of one power of two a group of heads."""
    q = q.float().unflatten(1, (kv_heads, -1))
    amax = q.abs().amax((-1, -2), keepdim=True)
    step = torch.ldexp(torch.ones_like(amax), torch.frexp(amax)[1] - 7)
    step = torch.where(amax > 127 * step, 2 * step, step).clamp(min=LOWEST)
    return torch.round(q / step)


def block_places(s, j):
    """Page and part of block j (any shape with rows in front) of each row's request; out of range wherever j is."""
    c = s["case"]
    per = c["page"] // c["block"]
    at = s["indptr"][:-1].long()[s["q_req"].long()].view(-1, *([1] * (j.dim() - 1)))
    return s["indices"].long()[(at + j // per).clamp(0, s["indices"].numel() - 1)], j % per


def plain_select(s):
    c = s["case"]
    h, block, top = c["kv_heads"], c["block"], c["top"]
    n = s["q_kvlen"].long()
    have = (n + block - 1) // block
    width = max(-(-s["max_kvlen"] // block), top)
    a = in_steps(s["q"], h).double()
    parts = torch.cat([a.clamp(min=0).sum(2), a.clamp(max=0).sum(2)], -1).transpose(0, 1).contiguous()         # [h, rows, 2 d]: what meets the largest, the smallest
    # every request's blocks, and every row's products with all of them: whole numbers, exact in 64 bits
    reqs, per = s["indptr"].numel() - 1, c["page"] // block
    j = torch.arange(width, device=DEV)
    where = (s["indptr"][:-1].long()[:, None] + j // per).clamp(0, s["indices"].numel() - 1)
    pages = s["indices"].long()[where]
    bounds = s["bounds"][pages, :, j % per].flatten(-2).reshape(reqs * width, h, -1).permute(1, 2, 0).double().contiguous()
    whole = torch.bmm(parts, bounds).unflatten(2, (reqs, width))[:, torch.arange(n.numel(), device=DEV), s["q_req"].long()].transpose(0, 1)
    steps = s["steps"][pages, :, j % per].transpose(1, 2)[s["q_req"].long()]
    score = whole.float() * steps
    always = (j < FIRST) | (j >= have[:, None] - LAST)
    score = torch.where(always[:, None], torch.inf, score)
    score = torch.where((j >= have[:, None])[:, None], -torch.inf, score)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    chosen = torch.where(order < have[:, None, None], order, width).sort(-1).values
    return torch.where(chosen < width, chosen, -1).to(torch.int32)


def plain_attend(s):
    c, kv = s["case"], s["kv"]
    h, block = c["kv_heads"], c["block"]
    j = s["blocks"].long()
    page, part = block_places(s, j.clamp(min=0))
    token = torch.arange(block, device=DEV)
    slot = part[..., None] * block + token
    head = torch.arange(h, device=DEV)[None, :, None, None]
    rows = j.shape[0]
    k = kv[page[..., None], 0, slot, head].float().reshape(rows * h, -1, c["dim"])
    q = s["q"].float().reshape(rows * h, -1, c["dim"])
    z = torch.bmm(q, k.transpose(1, 2).contiguous()).unflatten(0, (rows, h)) * s["scale"]
    del k
    seen = ((j[..., None] >= 0) & (j[..., None] * block + token < s["q_kvlen"].long()[:, None, None, None])).flatten(2)
    z = torch.where(seen[:, :, None], z, -torch.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    v = kv[page[..., None], 1, slot, head].float().reshape(rows * h, -1, c["dim"])
    o = torch.bmm(p.reshape(rows * h, -1, p.shape[-1]), v).unflatten(0, (rows, h)) / p.sum(-1, keepdim=True)
    return o.reshape(rows, -1, c["dim"]).to(kv.dtype)


def run(s):
    c = s["case"]
    if own:
        from vox_serve_amd import block_attention as B
        if c["kind"] == "append":
            q, k, v = split_qkv(s)
            q_out = B.rope_append(q, k, v, s["kv"], s["cos_sin"], s["pos"], s["pages"], s["slots"], interleave=c["pairs"] == "neighbours",
                                  bounds=s["bounds"], steps=s["steps"], n_req=c["reqs"])
        elif c["kind"] == "select":
            return B.select_blocks(s["q"], s["bounds"], s["steps"], s["q_req"], s["q_kvlen"], s["indptr"], s["indices"], block=c["block"], top=c["top"],
                                   max_kvlen=s["max_kvlen"], first=FIRST, last=LAST, n_req=c["reqs"])
        else:
            return B.block_attention(s["q"], s["kv"], s["blocks"], s["q_req"], s["q_kvlen"], s["indptr"], s["indices"], block=c["block"], scale=s["scale"], n_req=c["reqs"])
    elif c["kind"] == "append":
        q_out = plain_append(s)
    elif c["kind"] == "select":
        return plain_select(s)
    else:
        return plain_attend(s)
    return dict(q=q_out, kv=s["kv"], bounds=s["bounds"], steps=s["steps"])


def work(case):
    rows, heads, h, d, block = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    if case["kind"] == "append":
        # q, k and v read and written once, a row's angles; the bounds of one row in `block`
        return dict(bytes=rows * (4 * d * (heads + 2 * h) + 4 * case["rot"] + 12) + rows // block * h * (2 * d + 4), flops=3 * rows * (heads + h) * case["rot"])
    blocks = case["reqs"] * 0.8 * case["ctx"] / block
    if case["kind"] == "select":
        have = min(0.8 if case["reqs"] > 1 else 1.0, 1.0) * case["ctx"] / block
        return dict(bytes=blocks * h * (2 * d + 4) + rows * (2 * heads * d + 4 * h * case["top"] + 8), flops=2 * rows * h * have * 2 * d)
    # a chunk's rows share their request's blocks
    tokens = min(rows * case["top"] * block, case["reqs"] * case["ctx"])
    return dict(bytes=tokens * h * d * 4 + rows * (4 * heads * d + 4 * h * case["top"] + 8), flops=4 * rows * heads * min(case["top"] * block, case["ctx"]) * d)


def exact(case, seed):
    s = prepare(case, seed)
    kv, h, d, block, page = s["kv"], case["kv_heads"], case["dim"], case["block"], case["page"]
    rows, group = case["rows"], case["heads"] // case["kv_heads"]
    if case["kind"] == "append":
        # each pair is a complex number, turned by one multiplication
        kv = kv.double()
        half, near = case["rot"] // 2, case["pairs"] == "neighbours"
        by = torch.view_as_complex(s["cos_sin"].double()[s["pos"].long()].contiguous())[:, None]

        def turned(x):
            x = x.double().clone()
            first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if near else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., first], x[..., second]) * by
            x[..., first], x[..., second] = z.real, z.imag
            return x
        q, k, v = split_qkv(s)
        at = (s["pages"].long() * page + s["slots"].long())
        keys, values = kv[:, 0].reshape(-1, h, d), kv[:, 1].reshape(-1, h, d)
        keys[at], values[at] = turned(k), v.double()
        return dict(q=turned(q), kv=torch.stack([keys, values], 1).reshape(-1, page, 2, h, d).transpose(1, 2), bounds=None, steps=None)
    indptr, indices, req, lens = (s[n].tolist() for n in ("indptr", "indices", "q_req", "q_kvlen"))
    table = torch.tensor(indices, device=DEV)
    out = []
    for i in range(rows):
        mine = table[indptr[req[i]]:indptr[req[i] + 1]]
        q = s["q"][i].double().reshape(h, group, 1, d)
        if case["kind"] == "attend":
            j = s["blocks"][i].long()
            t = (j[..., None] * block + torch.arange(block, device=DEV)).flatten(1)
            seen = (t < lens[i]) & (j >= 0).repeat_interleave(block, 1)
            t = t.clamp(0, lens[i] - 1)
            pick = kv[mine[t // page], :, t % page, torch.arange(h, device=DEV)[:, None]].double()       # [h, tokens, 2, d]
            z = (q * pick[:, None, :, 0]).sum(-1) * s["scale"]
            p = torch.softmax(z.masked_fill(~seen[:, None], -math.inf), -1)
            out.append((p[..., None] * pick[:, None, :, 1]).sum(2).reshape(-1, d))
            continue
        count, top = -(-lens[i] // block), case["top"]
        row = torch.full((h, top), -1, dtype=torch.int32, device=DEV)
        if count <= top:
            row[:, :count] = torch.arange(count, device=DEV, dtype=torch.int32)
        else:
            j = torch.arange(FIRST, count - LAST, device=DEV)
            place = mine[j * block // page], (j * block % page) // block
            bound, unit = s["bounds"][place[0], :, place[1]].transpose(0, 1).double(), s["steps"][place[0], :, place[1]].t()      # [h, blocks, 2, d], [h, blocks]
            unit_q = torch.exp2(torch.ceil(torch.log2(q.abs().amax((1, 2, 3)) / 127)).clamp(min=-100))[:, None, None, None]       # the smallest power of two that 127 of reach the largest
            a = torch.round(q / unit_q)
            value = torch.maximum(a * bound[:, None, :, 0], a * bound[:, None, :, 1]).sum((1, 3)).float() * unit
            best = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :top - FIRST - LAST] + FIRST
            ends = torch.cat([torch.arange(FIRST, device=DEV), torch.arange(count - LAST, count, device=DEV)]).expand(h, -1)
            row[:] = torch.cat([best, ends], 1).sort(1).values
        out.append(row)
    return torch.stack(out)
