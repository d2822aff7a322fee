"""Workloads of the frame-attention operators: rotary positions over (time, height, width), block means, block selection and
attention over the selected blocks.

A target frame's feature tokens look for what their holes hide among the tokens of the reference frames.  Feature maps of the
networks in this package have 16 x 16, 30 x 53, 60 x 106 or 64 x 64 positions, 128 to 512 channels (split into heads of 32 to 128)
and 4 to 60 reference frames, so one target frame faces up to 381,600 reference tokens.  Keys lie in blocks of 64 or 128 consecutive
tokens; a group of queries (one token, or a run of `q_block` tokens, with all query heads that share a key head) scores the blocks by
their mean key and attends to the best `top_k` of them.

`run(state)` is one call of one operator: in plain torch operations, or (own = True) through master_thesis_amd.utils.attention."""
import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------------------------------------- cases
def _rotate(name, **kw):
    return {"name": name, "op": "rotate", "dtype": "float32", "items": 1, "frames": 1, "height": 16, "width": 16, "axes": 3, "heads": 8, "dim": 64,
            "interleaved": False, "per_item": False, "first_frame": 0, "grad": False, **kw}


def _means(name, **kw):
    return {"name": name, "op": "means", "dtype": "float32", "items": 1, "keys": 1590, "kv_heads": 2, "dim": 64, "block": 64, "masked": True,
            "heads_first": False, **kw}


def _select(name, **kw):
    return {"name": name, "op": "select", "dtype": "bfloat16", "items": 1, "queries": 1590, "blocks": 249, "heads": 2, "kv_heads": 2, "dim": 64,
            "q_block": 64, "top_k": 32, **kw}


def _attend(name, **kw):
    return {"name": name, "op": "attend", "dtype": "bfloat16", "items": 1, "queries": 1590, "keys": 15900, "heads": 2, "kv_heads": 2, "dim": 64,
            "block": 64, "q_block": 64, "top_k": 32, "masked": True, "heads_first": False, "grad": False, **kw}


def listed():
    return [
        # the tokens of one 16 x 16 target map, 512 channels: the smallest call, all latency
        _rotate("rotate_target_f32"),
        # the keys of 32 targets with 10 reference maps of 30 x 53 each, 128 channels
        _rotate("rotate_refs_bf16", dtype="bfloat16", items=32, frames=10, height=30, width=53, heads=2),
        # a training step on 64 x 64 maps, 256 channels, adjacent pairs, each clip at its own time, far into a long video
        _rotate("rotate_train_f16", dtype="float16", items=16, frames=1, height=64, width=64, heads=2, dim=128, interleaved=True, per_item=True,
                first_frame=100000, grad=True),
        # the block summary of one newly decoded reference frame
        _means("means_frame_f32"),
        # the summaries of all reference maps of 32 targets, holes left out
        _means("means_refs_bf16", dtype="bfloat16", items=32, keys=15900),
        # every 64-token tile of a 30 x 53 target chooses 32 of its 249 blocks, 32 targets
        _select("select_tiles_bf16", items=32),
        # every token of a 64 x 64 target chooses its own blocks from 4 reference maps, for a group of four query heads
        _select("select_tokens_f32", dtype="float32", items=16, queries=4096, blocks=256, heads=4, kv_heads=1, q_block=1, top_k=16),
        # inference: 32 targets of 30 x 53 against their 10 visible reference maps
        _attend("attend_refs_bf16", items=32),
        # a training step on 60 x 106 maps with 10 references, 256 channels
        _attend("attend_train_bf16", items=4, queries=6360, keys=63600, dim=128, top_k=64, grad=True),
        # a training step in full precision on 64 x 64 maps with 4 references, no holes
        _attend("attend_train_f32", dtype="float32", items=2, queries=4096, keys=16384, heads=4, kv_heads=4, top_k=16, masked=False, grad=True),
        # one token against 60 kept frames of 60 x 106: eight query heads to a key head, pages of 128 tokens
        _attend("attend_one_f16", dtype="float16", items=4, queries=1, keys=381600, heads=16, kv_heads=2, dim=128, block=128, q_block=1, top_k=64,
                masked=False, heads_first=True),
        # every token with blocks of its own, eight query heads to a key head, an odd head size
        _attend("attend_tokens_bf16", queries=1590, heads=16, dim=72, q_block=1, top_k=12),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotate", "means", "select", "attend", "attend"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    dim = rng.choice([32, 40, 64, 72, 96, 128])
    if op == "rotate":
        c = _rotate("", dtype=dtype, items=_log(rng, 1, 32), frames=_log(rng, 1, 10), height=_log(rng, 4, 64), width=_log(rng, 4, 106),
                    axes=rng.choice([2, 3]), heads=rng.choice([1, 2, 4, 8]), dim=dim, interleaved=rng.random() < 0.5, per_item=rng.random() < 0.5,
                    first_frame=rng.choice([0, 17, 100000]), grad=rng.random() < 0.5)
        while c["items"] * c["frames"] * c["height"] * c["width"] * c["heads"] * dim > 32 * 15900 * 128:
            c["items"], c["height"] = max(1, c["items"] // 2), max(4, c["height"] // 2)
    elif op == "means":
        c = _means("", dtype=dtype, items=_log(rng, 1, 32), keys=_log(rng, 1, 15900), kv_heads=rng.choice([1, 2]), dim=dim if dim <= 64 else 64,
                   block=rng.choice([64, 128]), masked=rng.random() < 0.7, heads_first=rng.random() < 0.3)
    elif op == "select":
        kv, q_block, blocks = rng.choice([1, 2]), rng.choice([1, 16, 64, 128]), _log(rng, 24, 400)
        c = _select("", dtype=dtype, items=_log(rng, 1, 16), queries=_log(rng, 1, 4096), blocks=blocks, kv_heads=kv,
                    heads=kv * rng.choice([1, 2, 4]), dim=dim, q_block=q_block, top_k=_log(rng, 4, blocks // 4))
    else:
        kv = rng.choice([1, 2])
        group = rng.choice([1, 2, 8])
        q_block = rng.choice([1, 16, 64, 128])
        c = _attend("", dtype=dtype, items=_log(rng, 1, 4), queries=_log(rng, 1, 2000 if q_block > 1 else 300), keys=_log(rng, 1, 20000), kv_heads=kv,
                    heads=kv * group, dim=dim, block=rng.choice([64, 128]), q_block=q_block, top_k=_log(rng, 1, 24), masked=rng.random() < 0.7,
                    heads_first=rng.random() < 0.5, grad=rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _axes(case):
    """Channels of each axis: height and width get three eighths each, time the rest (two axes: a half each)."""
    d = case["dim"]
    if case["axes"] == 2:
        return (d // 4 * 2, d - d // 4 * 2)
    side = 3 * d // 16 * 2
    return (d - 2 * side, side, side)


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(DTYPES[dtype])


def _tokens(case, gen, count, heads, scale=1.0):
    if case.get("heads_first"):
        return _normal(gen, (case["items"], heads, count, case["dim"]), case["dtype"], scale).transpose(1, 2)
    return _normal(gen, (case["items"], count, heads, case["dim"]), case["dtype"], scale)


def _visibility(case, gen, count):
    """1 = visible: holes in runs of 16 tokens, and in long caches the first two blocks of the first clip hidden altogether."""
    if not case["masked"]:
        return None
    runs = (torch.rand((case["items"], -(-count // 16)), generator=gen, device=DEV) < 0.75).float()
    runs[:, 0] = 1
    v = runs.repeat_interleave(16, 1)[:, :count].contiguous()
    if count > 8 * case["block"]:
        v[0, :2 * case["block"]] = 0
    return v


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "rotate":
        t, h, w = case["frames"], case["height"], case["width"]
        grid = torch.stack(torch.meshgrid(torch.arange(t, device=DEV) + case["first_frame"], torch.arange(h, device=DEV), torch.arange(w, device=DEV),
                                          indexing="ij"), -1).reshape(t * h * w, 3).float()
        if case["axes"] == 2:
            grid = grid[:, 1:].contiguous()
        if case["per_item"]:   # each clip starts at its own frame (or row)
            shift = torch.randint(0, 240, (case["items"], 1, 1), generator=gen, device=DEV).float()
            grid = torch.cat([grid[None, :, :1] + shift, grid[None, :, 1:].expand(case["items"], -1, -1)], -1).contiguous()
        shape = (case["items"], t * h * w, case["heads"], case["dim"])
        s.update(x=_normal(gen, shape, case["dtype"]), positions=grid, sections=_axes(case))
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = _normal(gen, shape, case["dtype"])
    elif case["op"] == "means":
        s.update(k=_tokens(case, gen, case["keys"], case["kv_heads"]), visible=_visibility(case, gen, case["keys"]))
    elif case["op"] == "select":
        shape = (case["items"], case["kv_heads"], case["blocks"], case["dim"])
        means = torch.randn(shape, generator=gen, device=DEV) * 0.15 + torch.randn(shape[:3] + (1,), generator=gen, device=DEV) * 0.02
        counts = torch.randint(-8, 65, (case["items"], case["blocks"]), generator=gen, device=DEV, dtype=torch.int32).clamp_(min=0)   # some are all holes
        s.update(q=_tokens(case, gen, case["queries"], case["heads"]), means=means, counts=counts)
    else:
        nb = -(-case["keys"] // case["block"])
        groups = -(-case["queries"] // case["q_block"])
        s.update(q=_tokens(case, gen, case["queries"], case["heads"], 1.5), k=_tokens(case, gen, case["keys"], case["kv_heads"]),
                 v=_tokens(case, gen, case["keys"], case["kv_heads"]), visible=_visibility(case, gen, case["keys"]))
        # distinct blocks for every group, some chosen more often than others, in ascending order, -1 behind the last
        liking = torch.rand((case["items"], case["kv_heads"], groups, nb), generator=gen, device=DEV)
        liking += 0.5 * torch.rand((case["items"], case["kv_heads"], 1, nb), generator=gen, device=DEV)
        chosen = liking.argsort(-1, descending=True)[..., :case["top_k"]].sort(-1).values
        s["blocks"] = torch.nn.functional.pad(chosen, (0, case["top_k"] - chosen.shape[-1]), value=-1).to(torch.int32).contiguous()
        if case["grad"]:
            s["do"] = _normal(gen, (case["items"], case["queries"], case["heads"], case["dim"]), case["dtype"])
            s.update({n: s[n].requires_grad_(True) for n in ("q", "k", "v")})
    return s


# ------------------------------------------------------------------------------------------------- the operators, plain
def _plain_rotate(s, x, sign):
    """Pair i of axis a turns by p_a * 10000^(-2 i / d_a): angles in 64 bits, the products in 32."""
    exps = torch.cat([torch.arange(0, d, 2, dtype=torch.float64) / d for d in s["sections"]])
    axis = torch.cat([torch.full((d // 2,), i) for i, d in enumerate(s["sections"])]).to(x.device)
    ang = s["positions"].double()[..., axis] * (10000.0 ** -exps).to(x.device)      # ([items,] tokens, dim / 2)
    cos, sin = ang.cos().float().unsqueeze(-2), (sign * ang.sin()).float().unsqueeze(-2)
    if s["interleaved"]:
        first = torch.arange(0, s["dim"], 2, device=x.device)
        second = first + 1
    else:   # the two halves of each axis' channels
        starts = torch.cat([torch.full((d // 2,), sum(s["sections"][:i])) for i, d in enumerate(s["sections"])])
        within = torch.cat([torch.arange(d // 2) for d in s["sections"]])
        halves = torch.cat([torch.full((d // 2,), d // 2) for d in s["sections"]])
        first = (starts + within).to(x.device)
        second = first + halves.to(x.device)
    a, b = x[..., first].float(), x[..., second].float()
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y.to(x.dtype)


def _plain_means(s):
    k, block = s["k"], s["block"]
    b, n, h, d = k.shape
    nb = -(-n // block)
    see = torch.ones((b, n), device=k.device) if s["visible"] is None else s["visible"]
    see = torch.nn.functional.pad((see > 0.5), (0, nb * block - n)).view(b, nb, block)
    kk = torch.nn.functional.pad(k.double(), (0, 0, 0, 0, 0, nb * block - n)).view(b, nb, block, h, d)
    counts = see.sum(2, dtype=torch.int32)
    total = torch.where(see[..., None, None], kk, 0.0).sum(2)
    return (total / counts.clamp(min=1)[..., None, None]).float().transpose(1, 2).contiguous(), counts


def _plain_select(s):
    """Scores in 64 bits (a choice hangs on values that may lie close together); the best first, ties to the lower index."""
    q, means, counts, qb, top = s["q"], s["means"], s["counts"], s["q_block"], s["top_k"]
    b, n, h, d = q.shape
    hk, nb = means.shape[1], means.shape[2]
    groups = -(-n // qb)
    qq = torch.nn.functional.pad(q.double(), (0, 0, 0, 0, 0, groups * qb - n)).view(b, groups, qb, hk, h // hk, d).sum((2, 4))
    score = torch.matmul(qq.transpose(1, 2), means.double().transpose(2, 3).contiguous())
    score = torch.where((counts > 0)[:, None, None], score, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    best = torch.where(order.values[..., :top] > float("-inf"), order.indices[..., :top], nb).sort(-1).values
    best = torch.nn.functional.pad(best, (0, top - best.shape[-1]), value=nb)
    return torch.where(best < nb, best, -1).to(torch.int32)


def _plain_attend(s):
    """Softmax over the visible keys of the chosen blocks, gathered for every group of queries; zero where nothing is visible."""
    q, k, v, blocks, block, qb = s["q"], s["k"], s["v"], s["blocks"].long(), s["block"], s["q_block"]
    b, n, h, d = q.shape
    m, hk = k.shape[1], k.shape[2]
    g, groups, top = h // hk, blocks.shape[2], blocks.shape[3]
    pad = groups * qb - n

    def rows(t):   # (b, n, h, d) -> (b, hk, groups, g * qb, d)
        t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, pad)).view(b, groups, qb, hk, g, d)
        return t.permute(0, 3, 1, 4, 2, 5).reshape(b, hk, groups, g * qb, d)

    def back(t, like):
        t = t.view(b, hk, groups, g, qb, d).permute(0, 2, 4, 1, 3, 5).reshape(b, groups * qb, h, d)
        return t[:, :n].to(like.dtype).contiguous()

    at = blocks[..., None] * block + torch.arange(block, device=q.device)
    ok = (blocks[..., None] >= 0) & (at < m)
    at = at.clamp(0, m - 1).view(b, hk, groups, top * block)
    ok = ok.view(b, hk, groups, top * block)
    if s["visible"] is not None:
        ok = ok & (s["visible"] > 0.5)[torch.arange(b, device=q.device)[:, None, None, None], at]
    flat = at + m * torch.arange(b * hk, device=q.device).view(b, hk, 1, 1)
    whole = lambda t: t.float().transpose(1, 2).reshape(b * hk * m, d)   # noqa: E731
    kk, vv = whole(k)[flat], whole(v)[flat]
    qq = rows(q)
    p = torch.matmul(qq, kk.transpose(-1, -2)) * d ** -0.5
    p = torch.where(ok.unsqueeze(-2), p, float("-inf"))
    top_score = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top_score > float("-inf"), top_score, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p, vv)
    if not s["grad"]:
        return back(out, q)
    do = rows(s["do"])
    dvv = torch.matmul(p.transpose(-1, -2), do)
    ds = p * (torch.matmul(do, vv.transpose(-1, -2)) - (do * out).sum(-1, keepdim=True)) * d ** -0.5
    dq = torch.matmul(ds, kk)
    dkk = torch.matmul(ds.transpose(-1, -2), qq)
    del p, ds, kk, vv
    scatter = lambda t, like: torch.zeros((b * hk * m, d), device=q.device).index_add_(0, flat.view(-1), t.view(-1, d)) \
        .view(b, hk, m, d).transpose(1, 2).to(like.dtype).contiguous()   # noqa: E731
    return back(out, q), back(dq, q), scatter(dkk, k), scatter(dvv, v)


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        if s["op"] == "rotate":
            y = _plain_rotate(s, s["x"], 1.0)
            return (y, _plain_rotate(s, s["dy"], -1.0)) if s["grad"] else y
        if s["op"] == "means":
            return _plain_means(s)
        if s["op"] == "select":
            return _plain_select(s)
        return _plain_attend(s)


def _own(s):
    from master_thesis_amd.utils import attention
    if s["op"] == "rotate":
        y = attention.rotate_positions(s["x"], s["positions"], s["sections"], interleaved=s["interleaved"])
        return (y.detach(), *torch.autograd.grad(y, s["x"], s["dy"])) if s["grad"] else y
    if s["op"] == "means":
        return attention.block_means(s["k"], s["visible"], block=s["block"])
    if s["op"] == "select":
        return attention.select_blocks(s["q"], s["means"], s["counts"], s["top_k"], q_block=s["q_block"])
    out = attention.block_attention(s["q"], s["k"], s["v"], s["blocks"], s["visible"], block=s["block"], q_block=s["q_block"])
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])) if s["grad"] else out


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    d = case["dim"]
    if case["op"] == "rotate":
        tokens = case["frames"] * case["height"] * case["width"]
        elements = case["items"] * tokens * case["heads"] * d
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * elements * size) + 4 * case["axes"] * tokens * (case["items"] if case["per_item"] else 1), "flops": passes * 3 * elements}
    if case["op"] == "means":
        elements = case["items"] * case["keys"] * case["kv_heads"] * d
        nb = -(-case["keys"] // case["block"])
        return {"bytes": elements * size + 4 * case["items"] * (case["keys"] * case["masked"] + nb * (case["kv_heads"] * d + 1)), "flops": elements}
    b, hk, n, h = case["items"], case["kv_heads"], case["queries"], case["heads"]
    groups = -(-n // case["q_block"])
    if case["op"] == "select":
        nb = case["blocks"]
        return {"bytes": b * (n * h * d * size + 4 * nb * (hk * d + 1) + 4 * hk * groups * case["top_k"]),
                "flops": b * (n * h * d + 2 * hk * groups * nb * d)}
    nb = -(-case["keys"] // case["block"])
    seen = min(min(case["top_k"], nb) * case["block"], case["keys"])       # keys of one group
    touched = min(groups * seen, case["keys"])                              # keys that some group needs
    rows = b * n * h * d * size
    kv = b * hk * touched * d * size
    marks = 4 * b * (hk * groups * case["top_k"] + (touched if case["masked"] else 0))
    if case["grad"]:   # q, dout, out, dq; k, v, and dk, dv over every key
        return {"bytes": 4 * rows + 2 * kv + 2 * b * hk * case["keys"] * d * size + marks, "flops": 14 * b * h * n * seen * d}
    return {"bytes": 2 * rows + 2 * kv + marks, "flops": 4 * b * h * n * seen * d}


# ------------------------------------------------------------------------------------------------- the same from the definitions, in 64 bits
def _exact_rotate(s, x, conj):
    """Channel pairs as complex numbers, each multiplied by exp(i p theta)."""
    parts, at = [], 0
    for i, d in enumerate(s["sections"]):
        z = x[..., at:at + d].detach().double()
        z = torch.complex(z[..., 0::2], z[..., 1::2]) if s["interleaved"] else torch.complex(z[..., :d // 2], z[..., d // 2:])
        theta = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -2.0 * torch.arange(d // 2, dtype=torch.float64) / d).to(x.device)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), (-1 if conj else 1) * s["positions"][..., i:i + 1].double() * theta)
        z = z * turn.unsqueeze(-2)
        parts.append(torch.stack([z.real, z.imag], -1).flatten(-2) if s["interleaved"] else torch.cat([z.real, z.imag], -1))
        at += d
    return torch.cat(parts, -1)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rotate":
            y = _exact_rotate(s, s["x"], False)
            return (y, _exact_rotate(s, s["dy"], True)) if case["grad"] else y
        if case["op"] == "means":
            b, n, h, d = s["k"].shape
            nb = -(-n // case["block"])
            see = torch.ones((b, n), dtype=torch.float64, device=DEV) if s["visible"] is None else (s["visible"] > 0.5).double()
            where = (torch.arange(n, device=DEV) // case["block"])
            total = torch.zeros((b, nb, h, d), dtype=torch.float64, device=DEV).index_add_(1, where, s["k"].double() * see[..., None, None])
            counts = torch.zeros((b, nb), dtype=torch.float64, device=DEV).index_add_(1, where, see)
            return (total / counts.clamp(min=1)[..., None, None]).transpose(1, 2), None
        if case["op"] == "select":
            return None
        b, n, h, d = s["q"].shape
        m, hk = s["k"].shape[1:3]
        group = h // hk
        nb = -(-m // case["block"])
        out, dq = (torch.zeros((b, n, h, d), dtype=torch.float64, device=DEV) for _ in range(2))
        dk, dv = (torch.zeros((b, m, hk, d), dtype=torch.float64, device=DEV) for _ in range(2))
        for i in range(b):
            for j in range(hk):
                chosen = torch.zeros((s["blocks"].shape[2], nb + 1), dtype=torch.bool, device=DEV)
                chosen.scatter_(1, torch.where(s["blocks"][i, j] < 0, nb, s["blocks"][i, j]).long(), True)
                reach = chosen[:, :nb].repeat_interleave(case["q_block"], 0)[:n].repeat_interleave(case["block"], 1)[:, :m]
                if s["visible"] is not None:
                    reach = reach & (s["visible"][i] > 0.5)
                kk, vv = s["k"][i, :, j].double(), s["v"][i, :, j].double()
                for e in range(j * group, (j + 1) * group):
                    w = (s["q"][i, :, e].double() @ kk.T / d ** 0.5).masked_fill_(~reach, float("-inf"))
                    w = torch.softmax(w, -1).nan_to_num_(0.0)
                    out[i, :, e] = w @ vv
                    if case["grad"]:
                        do = s["do"][i, :, e].double()
                        dv[i, :, j] += w.T @ do
                        w *= (do @ vv.T).sub_((do * out[i, :, e]).sum(-1, keepdim=True)).div_(d ** 0.5)
                        dq[i, :, e] = w @ kk
                        dk[i, :, j] += w.T @ s["q"][i, :, e].double()
        return (out, dq, dk, dv) if case["grad"] else out
