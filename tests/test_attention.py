"""Frame attention (master_thesis_amd/utils/attention.py) against plain 64-bit implementations.

Tolerances are bounds of the kernels' own roundings, evaluated per element from the 64-bit reference (`h` = half a step of the type):
a rounding of the result costs h |y|; a 16-bit operand P or dS of a second product costs h per term, so h times the sum of the terms'
magnitudes; an fp32 sum of n terms at most (n + 2) 2^-24 times the sum of magnitudes."""
import pytest
import torch

from master_thesis_amd import TclError
from master_thesis_amd.utils import attention as A

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def inside(got, ref, tol, what):
    got, ref, tol = got.detach().cpu().double(), ref.double(), tol.double()
    assert got.shape == ref.shape, "%s: %s vs %s" % (what, tuple(got.shape), tuple(ref.shape))
    assert torch.isfinite(got).all(), "%s: not finite" % what
    off = (got - ref).abs() - tol
    if off.numel() and off.max() > 0:
        i = int(off.argmax())
        raise AssertionError("%s: %d of %d outside; got %r, reference %r, tolerance %r" % (
            what, int((off > 0).sum()), off.numel(), got.reshape(-1)[i].item(), ref.reshape(-1)[i].item(), tol.expand_as(ref).reshape(-1)[i].item()))


# ------------------------------------------------------------------------------------------------ plain forms, 64 bits
def ref_rotate(x, pos, sections, base, interleaved, sign=1.0):
    """-> (y, |a| + |b| of each element's pair)"""
    x = x.double()
    y, mag, at = x.clone(), torch.zeros_like(x), 0
    for i, d in enumerate(sections):
        for p in range(d // 2):
            ia, ib = (at + 2 * p, at + 2 * p + 1) if interleaved else (at + p, at + d // 2 + p)
            ang = sign * pos[..., i].double() * base ** (-2.0 * p / d)
            c, s = ang.cos().unsqueeze(-1), ang.sin().unsqueeze(-1)
            a, b = x[..., ia], x[..., ib]
            y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
            mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
        at += d
    return y, mag


def ref_reach(blocks, nq, nk, block, q_block, visible, b, hk):
    """bool (B,Hkv,Nq,Nk): may this query see this key?"""
    nb = -(-nk // block)
    reach = torch.zeros(b, hk, nq, nk, dtype=torch.bool)
    for i in range(b):
        for j in range(hk):
            for s in range(blocks.shape[2]):
                for e in blocks[i, j, s].tolist():
                    if 0 <= e < nb:
                        reach[i, j, s * q_block:(s + 1) * q_block, e * block:(e + 1) * block] = True
    return reach if visible is None else reach & (visible > 0.5)[:, None, None, :]


def ref_attention(q, k, v, reach, scale, do=None):
    """Dense, 64 bits.  -> dict of results, each with the magnitudes its tolerance needs"""
    dt = q.dtype
    h, d, nk = half(dt), q.shape[3], k.shape[1]
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    seen = reach.any(2)[..., None]                                            # contents of keys that nobody sees do not count
    k, v = (torch.where(seen, t, torch.zeros_like(t)).repeat_interleave(G, 1) for t in (k, v))
    m = reach.repeat_interleave(G, 1)
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~m, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.where(m, torch.exp(s - torch.where(lse > float("-inf"), lse, torch.zeros_like(lse))[..., None]), torch.zeros_like(s))
    out = p @ v
    # relative error of a probability: that of its score (fp32 sum of d products, one factor, exp2's own) and of the denominator
    es = ((d + 4) * U * (q.abs() @ k.abs().transpose(2, 3) * scale) + 8 * U).masked_fill(~m, 0)
    ep = es + es.amax(-1, keepdim=True) + (nk + 8) * U
    r = {"out": out, "lse": lse, "lse_tol": es.amax(-1) + (nk + 8) * U * (1 + lse.abs().nan_to_num(0, 0, 0))}
    h2 = 0.0 if dt == torch.float32 else h
    # fp16: a probability below 2^-14 keeps its absolute, not its relative step
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    r["out_tol"] = (p * (ep + h2) + tiny * m) @ v.abs() * 1.01 + h * out.abs() + (nk + 8) * U * (p @ v.abs())
    if do is not None:
        g = do.double().transpose(1, 2)
        dp = g @ v.transpose(2, 3)
        delta = (g * out).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        e_dp = (d + 4) * U * (g.abs() @ v.abs().transpose(2, 3)) + (g.abs() * (r["out_tol"] + (d + 4) * U * out.abs())).sum(-1, keepdim=True)
        e_ds = (p * e_dp + p * (dp - delta).abs() * (ep + 4 * U)) * scale + h2 * ds.abs() + (2.0 ** -25) * m * (dt == torch.float16)
        fold = lambda t: t.view(t.shape[0], -1, G, t.shape[2], t.shape[3]).sum(2)   # noqa: E731
        n2 = (G * q.shape[2] + 8) * U
        for name, w, e, y in (("dq", ds, e_ds, k), ("dk", ds.transpose(2, 3), e_ds.transpose(2, 3), q), ("dv", p.transpose(2, 3), (p * (ep + h2) + tiny * m).transpose(2, 3), g)):
            val, tol = w @ y, 1.01 * (e @ y.abs()) + (max(n2, (nk + 8) * U)) * (w.abs() @ y.abs())
            if name != "dq":
                val, tol = fold(val), fold(tol)
            r[name], r[name + "_tol"] = val.transpose(1, 2), (tol + h * val.abs()).transpose(1, 2)
    r["out"], r["out_tol"] = r["out"].transpose(1, 2), r["out_tol"].transpose(1, 2)
    return r


def tokens(g, b, n, h, d, dtype, layout="dense", scale=1.0):
    """-> (CPU tensor, GPU tensor) of the same values; layout: dense, heads_first, sliced (rows off 16 bytes), cache (part of a longer buffer)"""
    t = rnd(g, b, n, h, d, dtype=dtype, scale=scale)
    if layout == "heads_first":
        return t, t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    if layout == "sliced":
        w = torch.zeros(b, n, h, d + 3, dtype=dtype, device=DEV)
        w[..., 1:d + 1] = t.to(DEV)
        return t, w[..., 1:d + 1]
    if layout == "cache":
        w = torch.full((b, n + 9, h, d), float("nan"), dtype=dtype, device=DEV)
        w[:, 5:n + 5] = t.to(DEV)
        return t, w[:, 5:n + 5]
    return t, t.to(DEV)


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_refusals_without_gpu():
    x = torch.zeros(1, 2, 1, 8)
    for call in (lambda: A.rotate_positions(x, torch.zeros(2, 1), (8,)), lambda: A.block_means(x),
                 lambda: A.select_blocks(x, torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, dtype=torch.int32), 1),
                 lambda: A.block_attention(x, x, x, torch.zeros(1, 1, 1, 1, dtype=torch.int32))):
        with pytest.raises(TclError, match="GPU only"):
            call()


def test_c_entries_refuse_without_gpu():
    """Shape, argument and workspace errors come from the host, before anything is launched."""
    import ctypes
    from master_thesis_amd import _lib
    lib = _lib.lib()
    one, off = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
    sec = (ctypes.c_int32 * 2)(4, 4)
    rot = lambda x=one, n=2, d=8, sections=sec, ns=2, base=1e4, dt=0: lib.tcl_rotate_positions(   # noqa: E731
        x, 16, 8, 8, one, 0, 0, one, 16, 8, 8, 1, n, 1, d, sections, ns, base, 0, 0, dt, None)
    assert rot(n=0) == 0
    assert rot(d=7) == 5 and rot(d=258) == 5 and rot(dt=3) == 5
    assert rot(sections=(ctypes.c_int32 * 2)(4, 6)) == 1 and rot(sections=(ctypes.c_int32 * 2)(3, 5)) == 1
    assert rot(ns=5) == 2 and rot(base=0.0) == 2 and rot(base=float("inf")) == 2 and rot(base=float("nan")) == 2
    assert rot(x=None) == 2 and rot(x=off) == 2
    means = lambda k=one, n=64, d=8, block=64, st=8: lib.tcl_block_means(k, 512, st, 8, None, one, one, 1, n, 1, d, block, 1, None)   # noqa: E731
    assert means(n=0) == 0 and means(d=12) == 5 and means(d=136) == 5 and means(block=96) == 5 and means(k=off) == 2 and means(st=12) == 2
    sel = lambda nb=4, top=1, d=8, hk=1, ws=one, wsb=1 << 20: lib.tcl_select_blocks(one, 16, 8, 8, one, one, one, 1, 2, 2, hk, d, nb, top, 1, 0, ws, wsb, None)   # noqa: E731
    assert sel(nb=16385) == 5 and sel(top=0) == 1 and sel(hk=3) == 1 and sel(d=9) == 5 and sel(nb=600, wsb=8) == 3 and sel(nb=600, ws=None) == 3
    fwd = lambda q=one, nk=64, d=8, top=1, block=64, qb=1, hk=1, wsb=0, dt=0, b=1, lo=None: lib.tcl_block_attention_fwd(   # noqa: E731
        q, 16, 8, 8, one, 512, 8, 8, one, 512, 8, 8, None, one, one, 16, 8, 8, lo, None, b, 2, nk, 2, hk, d, top, block, qb, 1.0, dt, one, wsb, None)
    assert fwd(b=0) == 0
    assert fwd(d=4) == 5 and fwd(d=136) == 5 and fwd(top=2049) == 5 and fwd(block=32) == 5 and fwd(nk=64 * 65537) == 5 and fwd(dt=9) == 5
    assert fwd(hk=3) == 1 and fwd(qb=0) == 1 and fwd(q=off) == 2 and fwd(lo=off) == 2 and fwd(q=None) == 2 and fwd(nk=1 << 16, top=100) == 3
    need = lib.tcl_block_attention_bwd_workspace_bytes(1, 2, 64, 2, 1, 8, 1, 64, 1)
    bwd = lambda wsb, go=one: lib.tcl_block_attention_bwd(go, 16, 8, 8, one, 16, 8, 8, one, 512, 8, 8, one, 512, 8, 8, None, one, one, 16, 8, 8, None, one,   # noqa: E731
                                                          None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, 1, 2, 64, 2, 1, 8, 1, 64, 1, 1.0, 0, one, wsb, None)
    assert bwd(need - 1) == 3 and bwd(need, go=None) == 2
    assert lib.tcl_block_attention_fwd_workspace_bytes(1, 1, 1 << 20, 8, 1, 128, 64, 128, 1) > 256     # few rows, many keys: split


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(1, 2, 2, 8, device=DEV)
    k = torch.zeros(1, 70, 1, 8, device=DEV)
    pos = torch.zeros(2, 1, device=DEV)
    bl = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=DEV)
    means, counts = A.block_means(k)
    for exc, call in [
        (ValueError, lambda: A.rotate_positions(x, pos, (7,))), (ValueError, lambda: A.rotate_positions(x, pos, (10,))), (ValueError, lambda: A.rotate_positions(x, pos, ())),
        (ValueError, lambda: A.rotate_positions(x, torch.zeros(3, 1, device=DEV), (8,))), (TclError, lambda: A.rotate_positions(x, pos.double(), (8,))),
        (ValueError, lambda: A.rotate_positions(x, pos, (8,), base=-1.0)), (TclError, lambda: A.rotate_positions(x, pos.clone().requires_grad_(True), (8,))),
        (TclError, lambda: A.rotate_positions(x.double(), pos, (8,))), (ValueError, lambda: A.rotate_positions(x[0], pos, (8,))),
        (TclError, lambda: A.rotate_positions(x, pos.cpu(), (8,))),
        (ValueError, lambda: A.block_means(k[..., :4])), (ValueError, lambda: A.block_means(k, block=32)), (ValueError, lambda: A.block_means(k, torch.ones(1, 69, device=DEV))),
        (TclError, lambda: A.block_means(k, torch.ones(1, 70, device=DEV, dtype=torch.int32))),
        (ValueError, lambda: A.select_blocks(x, means, counts, 0)), (ValueError, lambda: A.select_blocks(x, means, counts, 1, q_block=0)),
        (TclError, lambda: A.select_blocks(x, means.half(), counts, 1)), (ValueError, lambda: A.select_blocks(x, means, counts[:, :1], 1)),
        (ValueError, lambda: A.select_blocks(x, means.expand(1, 3, 2, 8), counts, 1)),
        (TclError, lambda: A.select_blocks(x, torch.zeros(1, 1, 16385, 8, device=DEV), torch.zeros(1, 16385, dtype=torch.int32, device=DEV), 1)),
        (TclError, lambda: A.block_attention(x, k.half(), k.half(), bl)), (ValueError, lambda: A.block_attention(x, k, k[:, :69], bl)),
        (ValueError, lambda: A.block_attention(x, k, k, bl, q_block=1)), (TclError, lambda: A.block_attention(x, k, k, bl.long())),
        (ValueError, lambda: A.block_attention(x, k, k, bl, block=100)), (ValueError, lambda: A.block_attention(x, k, k, bl[..., :0])),
        (TclError, lambda: A.block_attention(x, k, k, bl.expand(1, 1, 1, 2049))), (ValueError, lambda: A.block_attention(x[:, :, :0], k, k, bl)),
        (ValueError, lambda: A.block_attention(x, k.expand(1, 70, 3, 8), k.expand(1, 70, 3, 8), bl)),
    ]:
        with pytest.raises(exc):
            call()


# ------------------------------------------------------------------------------------------------ rotary positions
ROTATE = [  # b, n, h, sections, d, interleaved, layout
    (1, 1, 1, (2,), 2, False, "dense"), (2, 17, 3, (16, 24, 24), 64, False, "dense"), (1, 257, 2, (16, 24, 24), 64, True, "heads_first"),
    (3, 5, 1, (12, 14, 14), 40, False, "dense"), (2, 33, 2, (6, 10), 24, False, "sliced"), (2, 33, 2, (6, 10), 24, True, "sliced"),
    (1, 70, 5, (32, 48, 48), 128, False, "cache"), (1, 9, 1, (64, 0, 64, 128), 256, True, "dense"), (4, 3, 7, (8, 2), 12, True, "heads_first"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,sections,d,interleaved,layout", ROTATE)
def test_rotate_positions(b, n, h, sections, d, interleaved, layout, dtype):
    g = torch.Generator().manual_seed(n * 31 + d)
    for positions in ("shared", "per item", "int32", "far"):
        pos = torch.randint(0, 300, (n, len(sections)) if positions == "shared" else (b, n, len(sections)), generator=g).float()
        if positions == "far":
            pos = pos + 1e6 + 0.25
        x, xd = tokens(g, b, n, h, d, dtype, layout)
        gy, gyd = tokens(g, b, n, h, d, dtype, layout)
        xd = xd.detach().requires_grad_(True)
        y = A.rotate_positions(xd, (pos.int() if positions == "int32" else pos).to(DEV), sections, 500.0, interleaved)
        assert y.dtype == dtype
        gx, = torch.autograd.grad(y, xd, gyd)
        # the pair's magnitude times: the fraction of a turn in fp32 (pi 2^-24 rad), sine / cosine (fp32: 4 2^-24; else the hardware's, 2^-18)
        # and the two products and their sum (3 2^-24)
        trig = 12 * U if dtype == torch.float32 else 2.0 ** -18
        for got, t, sign, what in ((y, x, 1.0, "y"), (gx, gy, -1.0, "gx")):
            ref, mag = ref_rotate(t, pos, sections, 500.0, interleaved, sign)
            inside(got, ref, half(dtype) * ref.abs() + (trig + 2 * half(dtype) * trig) * mag, "%s %s" % (what, positions))
        rest = sum(sections)
        assert torch.equal(y[..., rest:].cpu(), x[..., rest:])


@pytest.mark.gpu
def test_rotate_leaves_other_channels_alone_and_turns_back():
    g = torch.Generator().manual_seed(3)
    x = rnd(g, 1, 6, 2, 16).to(DEV)
    x[..., 12:] = float("nan")
    x[..., 13] = float("inf")
    pos = torch.arange(6.0, device=DEV)[:, None]
    y = A.rotate_positions(x, pos, (12,))
    assert torch.equal(y[..., 12:].isnan(), x[..., 12:].isnan()) and torch.equal(y[..., 13], x[..., 13]) and torch.isfinite(y[..., :12]).all()
    back = A.rotate_positions(y, -pos, (12,))
    inside(back[..., :12], x[..., :12].cpu(), torch.full((1,), 40 * U * 8), "back")
    assert torch.equal(y[:, :1, :, :12], x[:, :1, :, :12])                       # position 0 turns nothing
    e = A.rotate_positions(x[:, :1].expand(1, 6, 2, 16), pos * 0 + 2, (12,))      # broadcast input
    assert torch.equal(e[:, 0, :, :12], e[:, 5, :, :12])
    assert A.rotate_positions(x[:, :0], pos[:0], (12,)).shape == (1, 0, 2, 16)
    p = A.frame_positions(2, 3, 4, DEV, first_frame=7)
    assert p.shape == (24, 3) and p[23].tolist() == [8, 2, 3] and p[5].tolist() == [7, 1, 1]


# ------------------------------------------------------------------------------------------------ block means
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,d,block,layout", [(1, 1, 1, 8, 64, "dense"), (2, 64, 2, 64, 64, "dense"), (1, 65, 3, 40, 64, "heads_first"), (2, 300, 1, 128, 128, "cache"),
                                                  (1, 1000, 2, 72, 128, "sliced"), (3, 127, 1, 96, 128, "dense")])
def test_block_means(b, n, h, d, block, layout, dtype):
    g = torch.Generator().manual_seed(n + d)
    k, kd = tokens(g, b, n, h, d, dtype, layout)
    nb = -(-n // block)
    for masked in (False, True):
        vis = (torch.rand(b, n, generator=g) < 0.5).float() if masked else torch.ones(b, n)
        if masked:
            vis[0, :block] = 0
            kd = torch.where(vis.to(DEV)[..., None, None] > 0.5, kd, torch.full_like(kd, float("nan")))
        means, counts = A.block_means(kd, vis.to(DEV) if masked else None, block)
        assert means.dtype == torch.float32 and counts.dtype == torch.int32
        for j in range(nb):
            sl = slice(j * block, (j + 1) * block)
            c = vis[:, sl].sum(1)
            total = (k[:, sl].double() * vis[:, sl, None, None].double()).sum(1)
            ref = total / c.clamp(min=1).double()[:, None, None]
            assert torch.equal(counts[:, j].cpu(), c.int())
            inside(means[:, :, j], ref, half(torch.float32) * ref.abs() * 1.001 + 1e-300, "block %d" % j)


# ------------------------------------------------------------------------------------------------ selection
def ref_select(q, means, counts, top, q_block):
    b, n, h, d = q.shape
    hk, nb = means.shape[1], means.shape[2]
    S = -(-n // q_block)
    out = torch.full((b, hk, S, top), -1, dtype=torch.int32)
    for i in range(b):
        for j in range(hk):
            for s in range(S):
                qs = q[i, s * q_block:(s + 1) * q_block, j * (h // hk):(j + 1) * (h // hk)].double().sum((0, 1))
                score = (means[i, j].double() @ qs).tolist()
                can = [x for x in range(nb) if counts[i, x] > 0 and score[x] > float("-inf")]
                best = sorted(sorted(can, key=lambda x: (-score[x], x))[:top])
                out[i, j, s, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,h,hk,d,nb,top,q_block,dtype", [
    (1, 1, 1, 1, 8, 1, 1, 1, torch.float32), (2, 5, 2, 2, 64, 15, 4, 1, torch.bfloat16), (1, 130, 4, 2, 40, 64, 9, 64, torch.float16),
    (2, 70, 2, 1, 72, 65, 70, 16, torch.float32), (1, 33, 8, 1, 128, 300, 24, 1, torch.bfloat16), (1, 20, 1, 1, 96, 513, 31, 3, torch.float32),
    (1, 3, 2, 1, 64, 1500, 64, 1, torch.float16), (1, 2, 1, 1, 32, 5000, 600, 2, torch.float32), (3, 200, 1, 1, 16, 257, 1, 1000, torch.float32),
    (1, 33, 4, 2, 128, 30, 5, 1, torch.float32), (2, 18, 8, 1, 96, 64, 12, 1, torch.float16)])
def test_select_blocks(b, n, h, hk, d, nb, top, q_block, dtype):
    g = torch.Generator().manual_seed(nb * 7 + n)
    q, means = rnd(g, b, n, h, d, dtype=dtype), rnd(g, b, hk, nb, d, scale=0.2)
    counts = torch.randint(-10, 65, (b, nb), generator=g, dtype=torch.int32).clamp(min=0)
    if nb >= 15:   # equal scores: the lower index wins
        means[:, :, nb // 2:nb // 2 + 4] = means[:, :, 2:3]
        counts[:, 2] = counts[:, nb // 2] = 64
    got = A.select_blocks(q.to(DEV), means.to(DEV), counts.to(DEV), top, q_block)
    assert torch.equal(got.cpu(), ref_select(q, means, counts, top, q_block))
    got = A.select_blocks(q.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), means.to(DEV), counts.to(DEV), top, q_block)
    assert torch.equal(got.cpu(), ref_select(q, means, counts, top, q_block))


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [40, 300, 700])
def test_select_ties_and_unusable_scores(nb):
    q, means = torch.zeros(1, 4, 1, 8, device=DEV), torch.randn(1, 1, nb, 8, device=DEV)
    counts = torch.ones(1, nb, dtype=torch.int32, device=DEV)
    q[0, 3] = 1.0
    means[0, 0, 5] = float("nan")
    means[0, 0, 6] = float("-inf")
    counts[0, 7] = 0
    got = A.select_blocks(q, means, counts, 9, 1)[0, 0]
    # zero queries: every finite mean scores 0 (0 * inf is NaN): the lowest indices
    assert got[0].tolist() == [0, 1, 2, 3, 4, 8, 9, 10, 11]
    assert got[1].tolist() == got[0].tolist()
    assert not set(got[3].tolist()) & {5, 6, 7}
    none = A.select_blocks(q, means, torch.zeros_like(counts), 3, 64)
    assert none.unique().tolist() == [-1]
    assert A.select_blocks(q, means[:, :, :0], counts[:, :0], 3, 64).unique().tolist() == [-1]
    assert A.select_blocks(q[:, :0], means, counts, 3, 64).shape == (1, 1, 0, 3)


# ------------------------------------------------------------------------------------------------ attention
def attention_case(g, b, nq, nk, hq, hk, d, block, q_block, top, dtype, masked, layout="dense", lists="ascending"):
    nb, S = -(-nk // block), -(-nq // q_block)
    q, qd = tokens(g, b, nq, hq, d, dtype, layout, 1.5)
    k, kd = tokens(g, b, nk, hk, d, dtype, layout)
    v, vd = tokens(g, b, nk, hk, d, dtype, layout)
    blocks = torch.full((b, hk, S, top), -1, dtype=torch.int32)
    for i in range(b):
        for j in range(hk):
            for s in range(S):
                pick = torch.randperm(nb, generator=g)[:top]
                if lists == "ascending":
                    blocks[i, j, s, :len(pick)] = pick.sort().values.int()
                else:   # out of order, with repeats and with indices that are no block
                    row = torch.cat([pick, pick[:2], torch.tensor([nb, -5, 2 ** 31 - 1, -2 ** 31])]).int()
                    blocks[i, j, s] = row[torch.randperm(len(row), generator=g)][:top]
    vis = None
    if masked:
        vis = (torch.rand(b, nk, generator=g) < 0.6).float()
        vis[0, :min(nk, 2 * block)] = 0
        hidden = (vis < 0.5).to(DEV)[..., None, None]
        kd = torch.where(hidden, torch.full_like(kd, float("nan")), kd)   # whatever lies in a hole must not matter
        vd = torch.where(hidden, torch.full_like(vd, float("inf")), vd)
    return (q, k, v), (qd, kd, vd), blocks, vis


ATTEND = [  # b, nq, nk, hq, hk, d, block, q_block, top, masked, layout, lists
    (1, 1, 1, 1, 1, 8, 64, 1, 1, False, "dense", "ascending"),
    (1, 1, 700, 8, 1, 64, 64, 1, 9, False, "heads_first", "ascending"),       # one token, split over its keys
    (2, 1, 1500, 16, 2, 128, 128, 1, 12, True, "cache", "mixed"),
    (2, 100, 300, 2, 2, 64, 64, 64, 3, True, "dense", "ascending"),
    (1, 130, 513, 4, 2, 40, 64, 64, 5, False, "heads_first", "mixed"),
    (1, 65, 200, 3, 1, 72, 128, 16, 2, True, "sliced", "ascending"),
    (2, 33, 129, 2, 1, 96, 64, 5, 3, True, "cache", "mixed"),
    (1, 300, 260, 1, 1, 128, 64, 300, 5, True, "dense", "ascending"),
    (1, 40, 640, 8, 1, 32, 64, 1, 4, False, "dense", "ascending"),             # every token with blocks of its own
    (1, 70, 190, 24, 1, 16, 64, 1, 2, True, "dense", "mixed"),
    (2, 64, 64, 1, 1, 64, 64, 128, 4, False, "dense", "ascending"),            # more choices than blocks, groups beyond the end
    (2, 70, 20, 2, 1, 64, 128, 16, 3, False, "dense", "ascending"),            # the last block of 128 ends in its first half
    (1, 1, 150, 8, 2, 128, 128, 1, 2, True, "heads_first", "mixed"),
    (1, 65, 300, 1, 1, 32, 128, 64, 3, True, "dense", "ascending"),
    (1, 600, 530, 4, 2, 128, 64, 64, 9, True, "dense", "ascending"),           # more than 2^20 scores: operands of the gradients in one part
    (1, 1100, 500, 2, 1, 64, 64, 16, 8, False, "heads_first", "mixed"),
    (2, 300, 1000, 2, 2, 96, 128, 100, 8, True, "cache", "mixed"),
    (1, 3000, 100, 8, 1, 32, 64, 64, 2, True, "dense", "ascending"),           # few keys, many rows: their gradients are split
    (2, 700, 70, 2, 2, 128, 128, 16, 1, False, "heads_first", "mixed"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ATTEND)
def test_block_attention(case, dtype):
    b, nq, nk, hq, hk, d, block, q_block, top, masked, layout, lists = case
    g = torch.Generator().manual_seed(nq * 1000 + nk + d)
    (q, k, v), dev, blocks, vis = attention_case(g, b, nq, nk, hq, hk, d, block, q_block, top, dtype, masked, layout, lists)
    do = rnd(g, b, nq, hq, d, dtype=dtype)
    reach = ref_reach(blocks, nq, nk, block, q_block, vis, b, hk)
    r = ref_attention(q, k, v, reach, d ** -0.5, do)
    leaves = [t.detach().requires_grad_(True) for t in dev]
    visd = None if vis is None else vis.to(DEV)
    out, lse = A.block_attention(*leaves, blocks.to(DEV), visd, block, q_block, return_lse=True)
    assert out.dtype == dtype and not lse.requires_grad
    inside(out, r["out"], r["out_tol"], "out")
    nothing = torch.isinf(r["lse"])
    assert torch.equal(torch.isinf(lse.cpu()), nothing)
    inside(lse.cpu().masked_fill(nothing, 0.0), r["lse"].masked_fill(nothing, 0.0), r["lse_tol"], "lse")
    grads = torch.autograd.grad(out, leaves, do.to(DEV))
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert got.dtype == dtype
        inside(got, r[name], r[name + "_tol"], name)
    again = torch.autograd.grad(A.block_attention(*leaves, blocks.to(DEV), visd, block, q_block), leaves, do.to(DEV))
    assert all(torch.equal(x, y) for x, y in zip(grads, again)), "the same inputs, other bits"
    with torch.no_grad():
        assert torch.equal(A.block_attention(*dev, blocks.to(DEV), None if vis is None else visd > 0.5, block, q_block), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.0, -0.7, 0.0])
@pytest.mark.parametrize("q_block", [1, 64])
def test_scores_that_rise_and_scales(q_block, scale, dtype):
    """Scores that climb by 60 along the keys, in small and large steps (a running maximum that moves all the time), and scales of any
    sign.  A negative scale is that of the turned queries."""
    g = torch.Generator().manual_seed(23)
    b, nq, nk, hq, hk, d = 1, 64, 700, 2, 1, 64
    u = rnd(g, d)
    u = u / u.norm()
    steps = torch.rand(nk, generator=g) * (torch.rand(nk, generator=g) < 0.1)
    ramp = steps.cumsum(0) / steps.sum() * 60 * (1 if scale >= 0 else -1)
    q = (u + rnd(g, b, nq, hq, d, scale=0.02)).to(dtype)
    k = (ramp[:, None, None] * u + rnd(g, b, nk, hk, d, scale=0.1)).to(dtype)
    v, do = rnd(g, b, nk, hk, d, dtype=dtype), rnd(g, b, nq, hq, d, dtype=dtype)
    vis = (torch.rand(b, nk, generator=g) < 0.8).float()
    groups = -(-nq // q_block)
    blocks = torch.arange(11).int().expand(b, hk, groups, 11).contiguous()
    reach = ref_reach(blocks, nq, nk, 64, q_block, vis, b, hk)
    sign = -1 if scale < 0 else 1
    r = ref_attention(sign * q, k, v, reach, abs(scale), do)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out, lse = A.block_attention(*leaves, blocks.to(DEV), vis.to(DEV), 64, q_block, scale=scale, return_lse=True)
    inside(out, r["out"], r["out_tol"], "out")
    inside(lse, r["lse"], r["lse_tol"], "lse")
    dq, dk, dv = torch.autograd.grad(out, leaves, do.to(DEV))
    inside(dq, sign * r["dq"], r["dq_tol"], "dq")
    inside(dk, r["dk"], r["dk_tol"], "dk")
    inside(dv, r["dv"], r["dv_tol"], "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nk,d", [(2, 128), (3, 64), (5, 128), (16, 128), (200, 32)])
def test_gradients_of_few_keys(nk, d, dtype):
    """With few keys, rowsum(dout o out) nearly cancels against its terms: the roundings that are allowed are those of the
    probabilities and the score gradients as operands and that of the result, NOT that of the forward's output.  A rounding is off by at most
    h of its value, by h / sqrt(3) of it or less in the square mean, and the roundings are independent: the squares of the errors
    of a whole tensor add up to the sum of the variances."""
    g = torch.Generator().manual_seed(nk + d)
    nq, h = 512, half(dtype)
    q, k, v, do = rnd(g, 1, nq, 1, d, dtype=dtype, scale=1.5), rnd(g, 1, nk, 1, d, dtype=dtype), rnd(g, 1, nk, 1, d, dtype=dtype), rnd(g, 1, nq, 1, d, dtype=dtype)
    top = -(-nk // 64)
    blocks = torch.arange(top).int().expand(1, 1, nq // 64, top).contiguous()
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(A.block_attention(*leaves, blocks.to(DEV)), leaves, do.to(DEV))
    Q, K, V, G = (t[0, :, 0].double() for t in (q, k, v, do))
    c = d ** -0.5
    P = torch.softmax(Q @ K.T * c, -1)
    dP = G @ V.T
    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * c
    of_delta = (P * dP).square().sum(-1, keepdim=True) * c * c
    for name, x, want, var in (("dq", got[0], dS @ K, dS.square() @ K.square() + of_delta * (P @ K).square()),
                               ("dk", got[1], dS.T @ Q, dS.square().T @ Q.square() + (P.square() * of_delta).T @ Q.square()),
                               ("dv", got[2], P.T @ G, P.square().T @ G.square())):
        bound = (h / 3 ** 0.5) * (want.square() + var).sum().sqrt().item()
        err = (x[0, :, 0].double().cpu() - want).norm().item()
        assert err <= bound, (name, err, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_block", [1, 64])
def test_the_longest_list_of_blocks(q_block, dtype):
    """2,048 chosen blocks of 2,100, the widest head: the most shared memory that a call can ask for."""
    g = torch.Generator().manual_seed(2048 + q_block)
    nq, nb, top, d = 40, 2100, 2048, 128
    nk = nb * 64 - 5
    (q, k, v), dev, blocks, vis = attention_case(g, 1, nq, nk, 1, 1, d, 64, q_block, top, dtype, True, "dense", "mixed")
    do = rnd(g, 1, nq, 1, d, dtype=dtype)
    r = ref_attention(q, k, v, ref_reach(blocks, nq, nk, 64, q_block, vis, 1, 1), d ** -0.5, do)
    leaves = [t.detach().requires_grad_(True) for t in dev]
    out = A.block_attention(*leaves, blocks.to(DEV), vis.to(DEV), 64, q_block)
    inside(out, r["out"], r["out_tol"], "out")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do.to(DEV))):
        inside(got, r[name], r[name + "_tol"], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_some_inputs(dtype):
    """Each input alone, keys that are the values, a cotangent without strides, the same graph twice: the bits of the whole step."""
    g = torch.Generator().manual_seed(91)
    (q, k, v), dev, blocks, vis = attention_case(g, 2, 90, 200, 4, 2, 40, 64, 32, 3, dtype, True)
    bl, vd = blocks.to(DEV), vis.to(DEV)
    leaves = [t.detach().requires_grad_(True) for t in dev]
    out = A.block_attention(*leaves, bl, vd, 64, 32)
    ones = torch.ones_like(out)
    whole = torch.autograd.grad(out, leaves, ones, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(whole, torch.autograd.grad(out.sum(), leaves, retain_graph=True)))
    assert all(torch.equal(x, y) for x, y in zip(whole, torch.autograd.grad(out, leaves, ones)))
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(dev)]
        assert torch.equal(torch.autograd.grad(A.block_attention(*some, bl, vd, 64, 32), some[i], ones)[0], whole[i])
    kv = torch.randn(2, 200, 2, 40, generator=g).to(dtype).to(DEV).requires_grad_(True)
    both = [leaves[0], kv, kv.detach().clone().requires_grad_(True)]
    _, dk, dv = torch.autograd.grad(A.block_attention(*both, bl, vd, 64, 32), both, ones)
    assert torch.equal(torch.autograd.grad(A.block_attention(leaves[0], kv, kv, bl, vd, 64, 32), kv, ones)[0], dk + dv)
    with pytest.raises(RuntimeError):
        grad = torch.autograd.grad(A.block_attention(*leaves, bl, vd, 64, 32), leaves[0], ones, create_graph=True)[0]
        torch.autograd.grad(grad.sum(), leaves[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_gradients_against_differences(dtype):
    """Central differences of the 64-bit plain form along random directions."""
    g = torch.Generator().manual_seed(5)
    (q, k, v), dev, blocks, vis = attention_case(g, 1, 70, 200, 2, 1, 24, 64, 32, 2, dtype, True)
    reach = ref_reach(blocks, 70, 200, 64, 32, vis, 1, 1)
    do = rnd(g, 1, 70, 2, 24, dtype=dtype)
    leaves = [t.detach().requires_grad_(True) for t in dev]
    grads = torch.autograd.grad(A.block_attention(*leaves, blocks.to(DEV), vis.to(DEV), 64, 32), leaves, do.to(DEV))
    value = lambda q, k, v: (ref_attention(q, k, v, reach, 24 ** -0.5)["out"] * do.double()).sum().item()   # noqa: E731
    r = ref_attention(q, k, v, reach, 24 ** -0.5, do)
    for i, name in enumerate(("dq", "dk", "dv")):
        args = [t.double() for t in (q, k, v)]
        u = rnd(g, *args[i].shape).double()
        eps = 1e-5
        plus, minus = [t.clone() for t in args], [t.clone() for t in args]
        plus[i] += eps * u
        minus[i] -= eps * u
        diff = (value(*plus) - value(*minus)) / (2 * eps)
        tol = (r[name + "_tol"] * u.abs()).sum().item() + 1e-6 * abs(diff) + 1e-7
        assert abs((grads[i].cpu().double() * u).sum().item() - diff) <= tol, name


@pytest.mark.gpu
def test_attention_empty_and_extreme():
    z = lambda *s: torch.zeros(*s, device=DEV)   # noqa: E731
    bl = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)   # noqa: E731
    assert A.block_attention(z(0, 4, 2, 8), z(0, 70, 1, 8), z(0, 70, 1, 8), bl(0, 1, 1, 2)).shape == (0, 4, 2, 8)
    assert A.block_attention(z(1, 0, 2, 8), z(1, 70, 1, 8), z(1, 70, 1, 8), bl(1, 1, 0, 2)).shape == (1, 0, 2, 8)
    q, k = torch.ones(1, 3, 2, 8, device=DEV, requires_grad=True), torch.zeros(1, 0, 1, 8, device=DEV, requires_grad=True)
    out, lse = A.block_attention(q, k, k, bl(1, 1, 1, 2), return_lse=True)
    assert out.abs().max() == 0 and torch.isneginf(lse).all()
    gq, gk = torch.autograd.grad(out.sum(), (q, k))
    assert gq.abs().max() == 0 and gk.shape == k.shape
    # nothing visible: zero rows, zero gradients, whatever the keys hold
    k = torch.full((1, 70, 1, 8), float("nan"), device=DEV, requires_grad=True)
    out = A.block_attention(q, k, k, bl(1, 1, 1, 2), torch.zeros(1, 70, device=DEV))
    grads = torch.autograd.grad(out.sum(), (q, k))
    assert out.abs().max() == 0 and all(t.abs().max() == 0 for t in grads)
    # large scores: the softmax neither overflows nor divides by zero
    for dtype in DTYPES:
        q, k = torch.full((1, 5, 1, 64), 30.0, device=DEV, dtype=dtype), torch.full((1, 130, 1, 64), -30.0, device=DEV, dtype=dtype)
        k[0, 77] = 30.0
        v = torch.arange(130.0, device=DEV)[None, :, None, None].expand(1, 130, 1, 64).to(dtype).contiguous()
        out = A.block_attention(q, k, v, torch.tensor([[[[0, 1, 2]]]], dtype=torch.int32, device=DEV), scale=1.0)
        assert (out == 77).all()
    # a NaN that is seen reaches the queries that see it, and no other
    v[0, 3] = float("nan")
    out = A.block_attention(q, k, v, torch.tensor([[[[0]], [[1]]]], dtype=torch.int32, device=DEV).view(1, 1, 2, 1), q_block=3)
    assert out[:, :3].isnan().all() and not out[:, 3:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_broadcast_inputs_and_partial_gradients(dtype):
    g = torch.Generator().manual_seed(8)
    q, k, v = (rnd(g, 1, n, h, 16, dtype=dtype).to(DEV) for n, h in ((20, 4), (90, 1), (90, 1)))
    bl = torch.tensor([0, 1], dtype=torch.int32, device=DEV).expand(3, 1, 1, 2)
    ke = k.clone().requires_grad_(True)
    out = A.block_attention(q.expand(3, 20, 4, 16), ke.expand(3, 90, 1, 16), v.expand(3, 90, 1, 16), bl)
    one = A.block_attention(q, k, v, bl[:1])
    assert all(torch.equal(out[i], one[0]) for i in range(3))
    gk, = torch.autograd.grad(out.float().sum(), ke)
    kd = k.clone().requires_grad_(True)
    gd, = torch.autograd.grad(A.block_attention(q, kd, v, bl[:1]).float().sum(), kd)
    inside(gk, 3 * gd.cpu().double(), 4 * half(dtype) * 3 * gd.cpu().double().abs() + 1e-30, "broadcast key gradient")
    for i in range(3):   # one gradient at a time
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        all_ = [t.clone().requires_grad_(True) for t in (q, k, v)]
        cot = rnd(g, 1, 20, 4, 16, dtype=dtype).to(DEV)
        single, = torch.autograd.grad(A.block_attention(*ts, bl[:1]), ts[i], cot)
        assert torch.equal(single, torch.autograd.grad(A.block_attention(*all_, bl[:1]), all_, cot)[i])
    with pytest.raises(RuntimeError):   # a second derivative is refused, not returned as zero
        gk, = torch.autograd.grad(A.block_attention(q, kd, v, bl[:1]).float().square().sum(), kd, create_graph=True)
        torch.autograd.grad(gk.float().sum(), kd)


@pytest.mark.gpu
def test_attention_under_autocast():
    g = torch.Generator().manual_seed(9)
    q, k = rnd(g, 1, 20, 2, 32).to(DEV).requires_grad_(True), rnd(g, 1, 90, 1, 32).to(DEV).requires_grad_(True)
    bl = torch.tensor([[[[0, 1]]]], dtype=torch.int32, device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = A.block_attention(q, k, k.half(), bl)
    assert out.dtype == torch.bfloat16
    gq, gk = torch.autograd.grad(out.float().sum(), (q, k))
    assert gq.dtype == gk.dtype == torch.float32
    assert torch.equal(out, A.block_attention(q.bfloat16(), k.bfloat16(), k.half().bfloat16(), bl))


# ------------------------------------------------------------------------------------------------ together
def frame_attention(q, k, v, pos_q, pos_k, sections, visible, top_k, q_block):
    q, k = A.rotate_positions(q, pos_q, sections), A.rotate_positions(k, pos_k, sections)
    means, counts = A.block_means(k, visible)
    blocks = A.select_blocks(q, means, counts, top_k, q_block)
    return A.block_attention(q, k, v, blocks, visible, q_block=q_block), blocks


def frame_inputs(seed, dtype, b=2, frames=3, h=9, w=11):
    g = torch.Generator().manual_seed(seed)
    n = h * w
    q, k, v = rnd(g, b, n, 4, 32, dtype=dtype, scale=1.5), rnd(g, b, frames * n, 2, 32, dtype=dtype), rnd(g, b, frames * n, 2, 32, dtype=dtype)
    vis = (torch.rand(b, frames * n, generator=g) < 0.7).float()
    pos = A.frame_positions(frames + 1, h, w, "cpu")
    return [t.to(DEV) for t in (q, k, v, pos[frames * n:], pos[:frames * n], vis)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_block", [1, 64])
def test_operators_together(dtype, q_block):
    sections = (8, 12, 12)
    q, k, v, pq, pk, vis = frame_inputs(1, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out, blocks = frame_attention(*leaves, pq, pk, sections, vis, 3, q_block)
    do = rnd(torch.Generator().manual_seed(2), *out.shape, dtype=dtype)
    grads = torch.autograd.grad(out, leaves, do.to(DEV))
    # the same chain in 64 bits; the rotated tensors are taken as the kernels rounded them, so that both sides attend to the same numbers
    qr, kr = (A.rotate_positions(t, p, sections).cpu() for t, p in ((q, pq), (k, pk)))
    for t, p, r in ((q, pq, qr), (k, pk, kr)):
        ref, mag = ref_rotate(t.cpu(), p.cpu(), sections, 10000.0, False)
        inside(r, ref, half(dtype) * ref.abs() + 2.0 ** -18 * mag, "rotated")
    means, counts = A.block_means(kr.to(DEV), vis)
    assert torch.equal(blocks.cpu(), ref_select(qr, means.cpu(), counts.cpu(), 3, q_block))
    n, nk = q.shape[1], k.shape[1]
    r = ref_attention(qr, kr, v.cpu(), ref_reach(blocks.cpu(), n, nk, 64, q_block, vis.cpu(), 2, 2), 32 ** -0.5, do)
    inside(out, r["out"], r["out_tol"], "out")
    inside(grads[2], r["dv"], r["dv_tol"], "dv")
    for name, got, p in (("dq", grads[0], pq), ("dk", grads[1], pk)):
        ref, _ = ref_rotate(r[name], p.cpu(), sections, 10000.0, False, -1.0)
        worst = r[name + "_tol"].amax(-1, keepdim=True) * 2 + 2 * half(dtype) * r[name].abs().amax(-1, keepdim=True) + 2.0 ** -17 * r[name].abs().amax(-1, keepdim=True)
        inside(got, ref, worst.expand_as(ref), name)


@pytest.mark.gpu
def test_together_on_another_stream_and_in_graphs():
    sections = (8, 12, 12)
    ins = [frame_inputs(s, torch.bfloat16) for s in (3, 4)]
    want = [frame_attention(*x[:5], sections, x[5], 3, 64)[0].clone() for x in ins]
    few = [frame_attention(x[0][:, :1], *x[1:3], x[3][:1], x[4], sections, x[5], 3, 1)[0].clone() for x in ins]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = frame_attention(*ins[0][:5], sections, ins[0][5], 3, 64)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want[0])
    # two graphs of the same calls, replayed in turn on changing inputs, eager work in between
    static = [[t.clone() for t in ins[0]] for _ in range(2)]
    graphs, outs = [], []
    for x in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((frame_attention(*x[:5], sections, x[5], 3, 64)[0], frame_attention(x[0][:, :1], *x[1:3], x[3][:1], x[4], sections, x[5], 3, 1)[0]))
        graphs.append(gr)
    for i in range(4):
        for j in range(2):
            src = ins[(i + j) % 2]
            for dst, t in zip(static[j], src):
                dst.copy_(t)
        for gr in graphs:
            gr.replay()
        eager = frame_attention(*ins[1][:5], sections, ins[1][5], 3, 64)[0]
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        for j in range(2):
            assert torch.equal(outs[j][0], want[(i + j) % 2]) and torch.equal(outs[j][1], few[(i + j) % 2])


@pytest.mark.gpu
def test_training_step_in_a_graph():
    q, k, v, pq, pk, vis = frame_inputs(6, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    bl = torch.arange(3, dtype=torch.int32, device=DEV).expand(2, 2, 2, 3).contiguous()
    do = torch.randn(q.shape, device=DEV).bfloat16()

    def step():
        x, y = A.rotate_positions(leaves[0], pq, (8, 12, 12)), A.rotate_positions(leaves[1], pk, (8, 12, 12))
        return torch.autograd.grad(A.block_attention(x, y, leaves[2], bl, vis), leaves, do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_cache_that_grows():
    """Serving: summaries of finished blocks are kept, a new frame appends; the answer is that of the whole cache."""
    g = torch.Generator().manual_seed(12)
    n, h, d = 128, 2, 64
    cache_k, cache_v = (torch.full((1, 5 * n, h, d), float("nan"), device=DEV, dtype=torch.float16) for _ in range(2))
    means, counts = torch.zeros(1, h, 10, d, device=DEV), torch.zeros(1, 10, dtype=torch.int32, device=DEV)
    for f in range(5):
        k, v = rnd(g, 1, n, h, d, dtype=torch.float16).to(DEV), rnd(g, 1, n, h, d, dtype=torch.float16).to(DEV)
        cache_k[:, f * n:(f + 1) * n], cache_v[:, f * n:(f + 1) * n] = k, v
        means[:, :, 2 * f:2 * f + 2], counts[:, 2 * f:2 * f + 2] = A.block_means(k)
        q = rnd(g, 1, 1, 8, d, dtype=torch.float16).to(DEV)
        got = A.block_attention(q, cache_k, cache_v, A.select_blocks(q, means, counts, 4, 1), q_block=1)      # blocks not written yet: count 0
        seen_k, seen_v = cache_k[:, :(f + 1) * n], cache_v[:, :(f + 1) * n]
        m, c = A.block_means(seen_k)
        bl = A.select_blocks(q, m, c, 4, 1)
        r = ref_attention(q.cpu(), seen_k.cpu(), seen_v.cpu(), ref_reach(bl.cpu(), 1, (f + 1) * n, 64, 1, None, 1, h), d ** -0.5)
        inside(got, r["out"], r["out_tol"], "frame %d" % f)


@pytest.mark.gpu
def test_long_cache_offsets_pass_31_bits():
    """Keys whose byte and element offsets lie beyond 2^31: the last blocks of a cache of 2^31 + elements."""
    n, h, d = (1 << 31) // 512 + 2048, 4, 128
    k = torch.zeros(1, n, h, d, device=DEV, dtype=torch.float16)
    g = torch.Generator().manual_seed(1)
    tail = rnd(g, 1, 300, h, d, dtype=torch.float16)
    k[:, n - 300:] = tail.to(DEV)
    nb = -(-n // 128)
    q = rnd(g, 1, 3, h, d, dtype=torch.float16)
    want = ref_attention(q, tail, tail, torch.ones(1, h, 3, 300, dtype=torch.bool), 0.05)
    vis = torch.zeros(1, n, device=DEV)
    vis[:, n - 300:] = 1
    bl = torch.arange(nb - 4, nb, dtype=torch.int32, device=DEV).expand(1, h, 1, 4)
    out = A.block_attention(q.to(DEV), k, k, bl, vis, block=128, scale=0.05)
    inside(out, want["out"], want["out_tol"], "out")
    m, c = A.block_means(k[:, :, :1], vis, 128)
    assert c[0, :nb - 4].abs().max() == 0 and int(c.sum()) == 300
    ref = tail[0, -(n % 128 or 128):, 0].double().mean(0)
    inside(m[0, 0, -1], ref, half(torch.float32) * ref.abs() + 1e-300, "means")


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def forward_mode_calls(dev):
    x, pos, bl = torch.randn(1, 2, 1, 8, device=dev), torch.zeros(2, 1, device=dev), torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=dev)
    return x, [("rotate_positions", lambda d, x: A.rotate_positions(d, pos, (8,))), ("rotate_positions", lambda d, x: A.rotate_positions(x, d[:, :, 0, :1], (8,))),
               ("block_attention", lambda d, x: A.block_attention(d, x, x, bl)), ("block_attention", lambda d, x: A.block_attention(x, d, x, bl)),
               ("block_attention", lambda d, x: A.block_attention(x, x, d, bl))]


def test_forward_mode_derivatives_are_refused():
    """A tangent is never dropped: not with requires_grad, not without, not under no_grad, not by torch.func."""
    from torch.autograd import forward_ad
    x, calls = forward_mode_calls("cpu")
    for what, call in calls:
        for grad in (False, True):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                with pytest.raises(NotImplementedError, match=what):
                    call(forward_ad.make_dual(x, torch.ones_like(x)), x)
        with pytest.raises(NotImplementedError, match=what):
            torch.func.jvp(lambda d: call(d, x), (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused_on_the_gpu():
    from torch.autograd import forward_ad
    x, calls = forward_mode_calls(DEV)
    for what, call in calls:
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match=what):
                call(forward_ad.make_dual(x, torch.ones_like(x)), x)
            plain = call(x, x)                                                    # in a level, without a tangent: as ever
        assert torch.equal(plain, call(x, x))


# ------------------------------------------------------------------------------------------------ scales that are no numbers
NO_SCALES = [float("nan"), float("inf"), -float("inf"), 3e38]


def test_c_entries_refuse_scales_that_are_not_finite():
    import ctypes
    from master_thesis_amd import _lib
    lib, one = _lib.lib(), ctypes.c_void_p(4096)
    for scale in NO_SCALES:
        assert lib.tcl_block_attention_fwd(one, 16, 8, 8, one, 512, 8, 8, one, 512, 8, 8, None, one, one, 16, 8, 8, None, None,
                                           1, 2, 64, 2, 1, 8, 1, 64, 1, scale, 0, one, 0, None) == 2
        assert lib.tcl_block_attention_bwd(one, 16, 8, 8, one, 16, 8, 8, one, 512, 8, 8, one, 512, 8, 8, None, one, one, 16, 8, 8, None, one,
                                           None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, 1, 2, 64, 2, 1, 8, 1, 64, 1, scale, 0, one, 1 << 20, None) == 2
        assert b"scale" in lib.tcl_last_error()


@pytest.mark.gpu
def test_scales_that_are_not_finite_are_refused():
    """(A NaN gave finite outputs: those of equal scores.)"""
    x, bl = torch.randn(1, 2, 1, 8, device=DEV, requires_grad=True), torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=DEV)
    for scale in NO_SCALES:
        for t in (x, x.detach()):
            with pytest.raises((ValueError, TclError), match="scale"):
                A.block_attention(t, t, t, bl, scale=scale)


# ------------------------------------------------------------------------------------------------ many groups
def test_c_entry_refuses_more_groups_than_the_grid_of_the_scores():
    import ctypes
    from master_thesis_amd import _lib
    lib, one = _lib.lib(), ctypes.c_void_p(4096)
    sel = lambda b, n, nb: lib.tcl_select_blocks(one, 16, 8, 8, one, one, one, b, n, 1, 1, 8, nb, 1, 1, 0, one, 1 << 60, None)   # noqa: E731
    assert sel(65536, 1, 513) == 1 and sel(1, 1 << 20, 513) == 1 and b"too many" in lib.tcl_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("b,n", [(1, (1 << 20) + 17), (70000, 1)])
def test_select_for_a_million_tokens_or_many_items(b, n):
    g = torch.Generator(device=DEV).manual_seed(4)
    q, means = torch.randn(b, n, 1, 8, device=DEV, generator=g), torch.randn(b, 1, 3, 8, device=DEV, generator=g)
    got = A.select_blocks(q, means, torch.ones(b, 3, dtype=torch.int32, device=DEV), 1, 1)
    score = (q[:, :, 0, None].double() * means[:, 0, None].double()).sum(-1)
    assert torch.equal(got[:, 0, :, 0], score.argmax(-1).int())


# ------------------------------------------------------------------------------------------------ the documented sequence
def documented():
    """The python blocks of the documents at the root that use the operators"""
    import pathlib
    import re
    texts = [p.read_text() for p in sorted(pathlib.Path(__file__).resolve().parent.parent.glob("*.md"))]
    return [b for t in texts for b in re.findall(r"```python\n(.*?)```", t, re.S) if "utils import attention as A" in b]


def test_documented_calls_fit_the_signatures():
    import ast
    import inspect
    assert documented()
    for block in documented():
        for n in ast.walk(ast.parse(block)):
            if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and isinstance(n.func.value, ast.Name) and n.func.value.id == "A":
                inspect.signature(getattr(A, n.func.attr)).bind(*n.args, **{k.arg: k.value for k in n.keywords})


@pytest.mark.gpu
def test_documented_sequence_runs():
    for block in documented():
        g = torch.Generator(device=DEV).manual_seed(1)
        maps = torch.randn(2, 128, 10, 30, 53, device=DEV, generator=g, dtype=torch.bfloat16)
        space = {"maps": maps, "heads": 2, "q": torch.randn(2, 1590, 2, 64, device=DEV, dtype=torch.bfloat16), "v": torch.randn(2, 15900, 2, 64, device=DEV, dtype=torch.bfloat16),
                 "visible": (torch.rand(2, 15900, device=DEV) < 0.8).float()}
        exec(block, space)
        assert space["out"].shape == (2, 1590, 2, 64) and torch.isfinite(space["out"]).all()
        assert torch.equal(space["maps"].view(2, 15900, 2, 64)[:, 1590 + 53 + 2, 1], maps[:, 64:, 1, 1, 2])      # frame 1, row 1, column 2
