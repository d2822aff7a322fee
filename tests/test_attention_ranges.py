"""Frame attention where the numbers themselves are hard: small and large cotangents, long sums, probabilities that lie binades apart.

Bounds are statistical, over whole tensors: a rounding is off by at most h of its value (half a step of the type), by h / sqrt(3) of it or less in the
square mean, the roundings are independent, and what the rounding of the exact result costs is computed, not estimated."""
import pytest
import torch

from master_thesis_amd.utils import attention as A
from .test_attention import DEV, half, rnd


def dense(q, k, v, do, scale):
    """One head whose queries see every key -> P, dP - delta, dS, in the type of the inputs"""
    p = torch.softmax(q @ k.T * scale, -1)
    dp = do @ v.T
    t = dp - (p * dp).sum(-1, keepdim=True)
    return p, t, p * t * scale


def gradients(q, k, v, do, q_block=64, scale=None):
    """of block_attention, every block chosen: q, k, v, do (N, D) on the CPU -> dq, dk, dv (N, D) in 64 bits"""
    top = -(-k.shape[0] // 64)
    blocks = torch.arange(top, device=DEV).int().expand(1, 1, -(-q.shape[0] // q_block), top).contiguous()
    leaves = [t.to(DEV)[None, :, None].requires_grad_(True) for t in (q, k, v)]
    out = A.block_attention(*leaves, blocks, q_block=q_block, scale=scale)
    return [t[0, :, 0].double() for t in torch.autograd.grad(out, leaves, do.to(DEV)[None, :, None])]


def own_rounding(x, dtype):
    return (x.to(dtype).double() - x).norm().item()


def check(name, got, want, var, dtype):
    """The error of the result's own rounding and that of one rounding of every operand (var: the squares of the terms, summed); a twentieth for the fp32 sums"""
    own, h = own_rounding(want, dtype), half(dtype)
    bound, err = 1.05 * (own ** 2 + h * h / 3 * var.sum().item()) ** 0.5, (got - want).norm().item()
    size = want.norm().item()
    assert err <= bound, "%s: error %.3g, own rounding %.3g, bound %.3g" % (name, err / size, own / size, bound / size)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("nk,d,q_block", [(4096, 128, 64), (1024, 64, 64), (1024, 64, 1), (200, 24, 64)])
def test_fp16_gradients_of_small_cotangents(nk, d, q_block, size):
    """A cotangent of 10^-3 and thousands of keys: the score gradients lie far below 2^-14, the results do not."""
    g = torch.Generator().manual_seed(nk + d)
    dtype, nq = torch.float16, 512
    q, k, v, do = rnd(g, nq, d, dtype=dtype, scale=1.5), rnd(g, nk, d, dtype=dtype), rnd(g, nk, d, dtype=dtype), rnd(g, nq, d, dtype=dtype, scale=size)
    dq, dk, dv = gradients(q, k, v, do, q_block)
    Q, K, V, G = (t.to(DEV).double() for t in (q, k, v, do))
    p, _, ds = dense(Q, K, V, G, d ** -0.5)
    check("dq", dq, ds @ K, ds.square() @ K.square(), dtype)
    check("dk", dk, ds.T @ Q, ds.square().T @ Q.square(), dtype)
    check("dv", dv, p.T @ G, p.square().T @ G.square(), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("nk", [5, 700])
def test_fp16_gradients_of_rows_of_all_sizes(nk):
    """Rows whose cotangents lie 20 binades apart in one call, values so large that with few keys a score gradient passes fp16's largest number; the
    keys (the queries) that it is multiplied by are small, and the results are ordinary numbers."""
    g = torch.Generator().manual_seed(nk)
    dtype, nq, d = torch.float16, 130, 64
    sizes = torch.exp2(-20 * torch.rand(nq, 1, generator=g)) * 1000
    v, do = rnd(g, nk, d, dtype=dtype, scale=1000), (rnd(g, nq, d) * sizes).to(dtype)
    for big, small, which in ((100.0, 0.01, "dq"), (0.01, 100.0, "dk")):
        q, k = rnd(g, nq, d, dtype=dtype, scale=big), rnd(g, nk, d, dtype=dtype, scale=small)
        p, _, ds = dense(*(t.double() for t in (q, k, v, do)), d ** -0.5)
        assert nk > 5 or ds.abs().max() > 2 ** 16
        dq, dk, _ = gradients(q, k, v, do)
        Q, K, ds = q.to(DEV).double(), k.to(DEV).double(), ds.to(DEV)
        if which == "dq":                                                         # every row for itself
            want, var = ds @ K, ds.square() @ K.square()
            for i in range(nq):
                check("dq %d" % i, dq[i], want[i], 15 * var[i], dtype)            # |sum of 5 errors|^2 <= 5 h^2 times the sum of squares
        else:
            check("dk", dk, ds.T @ Q, 15 * ds.square().T @ Q.square(), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_block", [1, 64])
def test_the_long_tail_of_a_row(q_block, dtype):
    """131,068 equal keys about 25 binades below four others: together they carry 2^-10 of the weight, and all of the output.  (512 groups: no split of the
    keys, in which the tail would be among its equals.)"""
    nk, d, groups = 2048 * 64, 8, 512
    q, k, v = torch.zeros(1, groups * q_block, 1, d, dtype=dtype), torch.zeros(1, nk, 1, d, dtype=dtype), torch.ones(1, nk, 1, d, dtype=dtype)
    q[..., 0] = 1.0
    k[0, [0, 16, 32, 48], 0, 0] = 17.47
    v[0, [0, 16, 32, 48]] = 0
    blocks = torch.arange(2048, device=DEV).int().expand(1, 1, groups, 2048).contiguous()
    out, lse = A.block_attention(q.to(DEV), k.to(DEV), v.to(DEV), blocks, q_block=q_block, scale=1.0, return_lse=True)
    s = k[0, :, 0, 0].double()
    want = (torch.softmax(s, 0) * v[0, :, 0, 0].double()).sum().item()
    # equal probabilities round alike (h), the result (h); a lane adds its equal ones up in 2^11 steps (2^-13)
    assert (out.double() - want).abs().max().item() <= (2 * half(dtype) + 2.0 ** -12) * want
    assert (lse.double() - torch.logsumexp(s, 0).item()).abs().max().item() <= 2.0 ** -13 + 32 * 2.0 ** -24


@pytest.mark.gpu
def test_fp16_value_gradient_of_an_unlikely_key():
    """P = 1.4 2^-33 and a cotangent of 2^14: dv is 45 of fp16's smallest steps."""
    q, k = torch.zeros(1, 1, 1, 8, dtype=torch.float16), torch.zeros(1, 2, 1, 8, dtype=torch.float16)
    q[..., 0], k[0, 0, 0, 0] = 1.0, 22.54
    v = torch.zeros_like(k).to(DEV).requires_grad_(True)
    out = A.block_attention(q.to(DEV), k.to(DEV), v, torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=DEV), scale=1.0)
    dv, = torch.autograd.grad(out, v, torch.full_like(out, 2.0 ** 14))
    want = torch.softmax(k[0, :, 0, 0].double(), 0) * 2.0 ** 14
    # half a step each for the operand and the result; the score's rounding (33 log2 units)
    assert (dv[0, 1, 0].double() - want[1].item()).abs().max().item() <= 2 * 2.0 ** -25 + 40 * 2.0 ** -24 * want[1].item()


@pytest.mark.gpu
@pytest.mark.parametrize("b,hk,nq,group,d,q_block", [(512, 1, 16000, 1, 8, 64), (128, 4, 2000, 8, 32, 64), (1, 1, 5000, 8, 128, 64), (1, 2, 4500, 8, 40, 1)])
def test_fp32_key_gradients_are_not_one_serial_sum(b, hk, nq, group, d, q_block):
    """Thousands of rows of every key, with key tiles enough for the whole GPU (no split of the rows) and with few.  A serial sum of n random terms has
    an error of about 0.4 sqrt(n / 2) u of its size (the partial sums' roundings, u = 2^-24): 36 u for 16,000.  Sums of at most 1,024 terms: 9 u.  The
    errors of the terms themselves are those of the same formulas in plain fp32 products, summed in blocks."""
    u, nk = 2.0 ** -24, 64
    g = torch.Generator(device=DEV).manual_seed(d)
    q, k, v, do = (torch.randn(b, n, h, d, device=DEV, generator=g) for n, h in ((nq, hk * group), (nk, hk), (nk, hk), (nq, hk * group)))
    visible = torch.ones(b, nk, device=DEV)
    visible[:, 40:50] = 0
    blocks = torch.zeros(b, hk, -(-nq // q_block), 1, dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    _, dk, dv = torch.autograd.grad(A.block_attention(*leaves, blocks, visible, q_block=q_block), leaves, do)
    assert dk[:, 40:50].abs().max() == 0 and dv[:, 40:50].abs().max() == 0
    seen = visible[0] > 0
    for i, j in ((0, 0), (b - 1, hk - 1)):
        rows = [t[i, :, j * group:(j + 1) * group].detach().reshape(-1, d) for t in (q, do)]
        keys = [t[i, seen, j].detach() for t in (k, v)]
        exact, plain = [], []
        for out, cast in ((exact, torch.float64), (plain, torch.float32)):
            Q, G, K, V = (t.to(cast) for t in rows + keys)
            p, _, ds = dense(Q, K, V, G, d ** -0.5)
            for w, y in ((ds, Q), (p, G)):
                out.append(sum(w[r:r + 512].T @ y[r:r + 512] for r in range(0, len(w), 512)))
        for name, got, want, near in zip(("dk", "dv"), (dk, dv), exact, plain):
            size = want.norm()
            err, floor = ((x.double() - want).norm().item() / size.item() / u for x in (got[i, seen, j], near))
            assert err <= 1.25 * (9.0 ** 2 + floor ** 2) ** 0.5, "%s: error %.1f u, that of the terms %.1f u" % (name, err, floor)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,d,q_block", [(32768, 16384, 64, 64), (512, 65536, 64, 1)])
def test_fp32_sums_over_many_keys(nq, nk, d, q_block):
    """Queries enough for the whole GPU (no split of the keys), thousands of keys each.  As above: a serial sum over 16,384 keys is off by 36 u of its size,
    of sums of 32 (few rows: 16 of each 64) by 0.4 sqrt(n / 64) u (few rows: 0.4 sqrt(n / 128) u, the query gradient's two halves as before).  The gradient's
    probabilities come from lse, 10 of 2^-20: roundings of 4.6 u, and of 3.2 u in log2 units, and those of the exponents, 3.2 u: 6.5 u."""
    u = 2.0 ** -24
    g = torch.Generator(device=DEV).manual_seed(nk)
    q, k, v, do = (torch.randn(1, n, 1, d, device=DEV, generator=g) for n in (nq, nk, nk, nq))
    top = nk // 64
    blocks = torch.arange(top, device=DEV).int().expand(1, 1, nq // q_block, top).contiguous()
    q.requires_grad_(True)
    out = A.block_attention(q, k, v, blocks, q_block=q_block)
    dq, = torch.autograd.grad(out, q, do)
    n = min(nq, 1024)
    sums = lambda w, y: sum(w[:, i:i + 512] @ y[i:i + 512] for i in range(0, nk, 512))   # noqa: E731
    results = []
    for cast in (torch.float64, torch.float32):
        Q, K, V, G = (t[0, :m, 0].detach().to(cast) for t, m in ((q, n), (k, nk), (v, nk), (do, n)))
        p, _, ds = dense(Q, K, V, G, d ** -0.5)
        results.append((sums(p, V), sums(ds, K)))
    for name, got, want, near in zip(("out", "dq"), (out, dq), *results):
        err, floor = (((x.double() - want).norm() / want.norm()).item() / u for x in (got[0, :n, 0].detach(), near))
        bound = 1.25 * (0.4 ** 2 * nk / 64 + 6.5 ** 2 + floor ** 2) ** 0.5
        assert err <= bound, "%s: error %.1f u, that of the terms %.1f u, bound %.1f u" % (name, err, floor, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,nq,nk,d", [(1, 300, 500, 64), (8, 300, 500, 64), (4, 4000, 100, 128), (64, 64, 3000, 96)])
def test_gradients_with_few_terms_are_exact_alone_and_in_a_batch(b, nq, nk, d, dtype):
    """Sums of few terms (queries or keys): the operands' roundings are no part of the error, whatever else is in the call.  What is left is the rounding of the
    result and that of the forward's probabilities, through rowsum(dout o out)."""
    g = torch.Generator().manual_seed(nk + d)
    h = half(dtype)
    q, k, v, do = (rnd(g, b, n, 1, d, dtype=dtype, scale=s) for n, s in ((nq, 1.5), (nk, 1), (nk, 1), (nq, 1)))
    top = -(-nk // 64)
    blocks = torch.arange(top, device=DEV).int().expand(b, 1, -(-nq // 64), top).contiguous()
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(A.block_attention(*leaves, blocks), leaves, do.to(DEV))
    for i in {0, b // 2, b - 1}:
        Q, K, V, G = (t[i, :, 0].to(DEV).double() for t in (q, k, v, do))
        c = d ** -0.5
        p, _, ds = dense(Q, K, V, G, c)
        delta = (p * (G @ V.T)).square().sum(-1, keepdim=True) * c * c           # variance of rowsum(dout o out) over h^2 / 3
        for name, x, want, var in (("dq", got[0], ds @ K, delta * (p @ K).square()), ("dk", got[1], ds.T @ Q, (p * p * delta).T @ Q.square()), ("dv", got[2], p.T @ G, None)):
            own = own_rounding(want, dtype)
            bound = 1.1 * (own ** 2 + (0 if var is None else h * h / 3 * var.sum().item())) ** 0.5
            err = (x[i, :, 0].double() - want).norm().item()
            assert err <= bound, "%s of item %d: %.3f times its own rounding, bound %.3f" % (name, i, err / own, bound / own)


@pytest.mark.gpu
@pytest.mark.parametrize("size,dtype", [(s, t) for s in (20.0, 100.0, 1e3, 1e4, 1e6, 1e8) for t in (torch.float32, torch.bfloat16, torch.float16)
                                        if s <= 1e6 or t != torch.float16])      # fp16: scores of up to 2 10^7
def test_gradients_under_large_scores(size, dtype):
    """Scores up to many times 10^8: the softmax is one key in the end, and its value gets the whole cotangent.  As exact as the same formulas in plain fp32
    products (scores of either side are rounded alike), and a few roundings: of P, its weight and the product."""
    g = torch.Generator().manual_seed(11)
    n, d = 1024, 64
    q, k, v, do = (rnd(g, n, d, dtype=dtype, scale=s) for s in (size ** 0.5, size ** 0.5, 1, 1))
    grads = gradients(q, k, v, do)
    results = []
    for cast in (torch.float64, torch.float32):
        Q, K, V, G = (t.to(DEV).to(cast) for t in (q, k, v, do))
        p, _, ds = dense(Q, K, V, G, d ** -0.5)
        results.append([t.double() for t in (ds @ K, ds.T @ Q, p.T @ G)])
    for name, got, want, near in zip(("dq", "dk", "dv"), grads, *results):
        if name != "dv" and (dtype != torch.float32 or size > 100):           # what the score's own rounding leaves of the differences
            continue
        err, floor = ((x - want).norm().item() / want.norm().item() for x in (got, near.to(dtype).double()))
        assert err <= 1.5 * floor + 4 * 2.0 ** -24, "%s: error %.3g, plain %.3g" % (name, err, floor)


@pytest.mark.gpu
@pytest.mark.parametrize("q_block", [1, 64])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 1.6e7), (torch.float16, 4e7), (torch.bfloat16, 1e9), (torch.float32, 1e9)])
def test_the_largest_scores(dtype, size, q_block):
    """All scores near `size`, one far above the rest: its value is the output, and its value's gradient the sum of the cotangents."""
    g = torch.Generator().manual_seed(13)
    n, d = 512, 64
    q, k = (torch.full((n, d), (8 * size / d) ** 0.5).to(dtype) for _ in range(2))
    k[77] *= 1.0625
    v, do = rnd(g, n, d, dtype=dtype), rnd(g, n, d, dtype=dtype)
    blocks = torch.arange(8, device=DEV).int().expand(1, 1, n // q_block, 8).contiguous()
    leaves = [t.to(DEV)[None, :, None].requires_grad_(True) for t in (q, k, v)]
    out = A.block_attention(*leaves, blocks, q_block=q_block)
    dv, = torch.autograd.grad(out, leaves[2], do.to(DEV)[None, :, None])
    h = half(dtype)
    want = v[77].to(DEV).double()
    assert ((out[0, :, 0].double() - want).abs() <= 2 * h * want.abs() + 2.0 ** -22).all()
    total = do.to(DEV).double().sum(0)
    near = (2 * h * do.to(DEV).double().square().sum(0).sqrt() * 6 + 2 * h * total.abs() + 2.0 ** -24 * n * do.to(DEV).double().abs().sum(0))
    assert ((dv[0, 77, 0].double() - total).abs() <= near).all()
    rest = dv[0, :, 0].clone()
    rest[77] = 0
    assert rest.abs().max() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_c_entries_with_lse_alone(dtype):
    """A caller that keeps nothing but lse: the gradients of the Python call, to the rounding of lse (6 at most: 2^-22, twice, of every probability)."""
    from master_thesis_amd import _lib, _ops
    g = torch.Generator().manual_seed(12)
    nq, nk, h, d = 70, 200, 2, 32
    q, do = (rnd(g, 1, nq, h, d, dtype=dtype).to(DEV) for _ in range(2))
    k, v = (rnd(g, 1, nk, h, d, dtype=dtype).to(DEV) for _ in range(2))
    blocks = torch.arange(4, device=DEV).int().expand(1, h, 2, 4).contiguous()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out, lse = A.block_attention(*leaves, blocks, return_lse=True)
    want = torch.autograd.grad(out, leaves, do)
    got_out, got_lse, lo = torch.empty_like(q), torch.full((h, nq), float("nan"), device=DEV), torch.empty_like(q)
    strides = [t for x in (q, k, v) for t in (x.data_ptr(), *_ops._strides(x))]
    sizes = (1, nq, nk, h, h, d, 4, 64, 64, d ** -0.5, _ops._DT[dtype])
    low = None if dtype == torch.float32 else lo.data_ptr()
    ws = torch.empty(_lib.lib().tcl_block_attention_bwd_workspace_bytes(*sizes[:9]) + (1 << 20), dtype=torch.uint8, device=DEV)
    tail = (ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    _lib.call("tcl_block_attention_fwd", *strides, None, blocks.data_ptr(), got_out.data_ptr(), *_ops._strides(q), low, got_lse.data_ptr(), *sizes, *tail)
    assert torch.equal(got_out, out) and torch.equal(got_lse, lse[0])
    got = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    _lib.call("tcl_block_attention_bwd", do.data_ptr(), *_ops._strides(do), *strides, None, blocks.data_ptr(), got_out.data_ptr(), *_ops._strides(q), low, got_lse.data_ptr(),
              *[t for x in got for t in (x.data_ptr(), *_ops._strides(x))], *sizes, *tail)
    for a, b in zip(got, want):
        assert (a.double() - b.double()).norm() <= (2.0 ** -20 + (0 if dtype == torch.float32 else half(dtype))) * b.double().norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nk,q_block", [(64, 3, 64), (64, 3, 1), (1, 4096, 1)])
def test_output_and_what_its_rounding_took(nq, nk, q_block, dtype):
    """Three equal keys are seen: probabilities of a third each, whose operands are exact.  What training keeps of the output next to it has to add up to the mean of
    the three values, also where that lies halfway between two numbers of the type."""
    from master_thesis_amd import _ops
    g = torch.Generator().manual_seed(nk)
    d, h = 128, half(dtype)
    v = rnd(g, 16, nk, 1, d, dtype=dtype).to(DEV)
    visible = torch.zeros(16, nk, device=DEV)
    at = [0, nk // 2, nk - 1]
    visible[:, at] = 1
    top = -(-nk // 64)
    blocks = torch.arange(top, device=DEV).int().expand(16, 1, -(-nq // q_block), top).contiguous()
    out, _, lo = _ops._attend(torch.zeros(16, nq, 1, d, dtype=dtype, device=DEV), torch.ones_like(v), v, blocks, visible, 64, q_block, 1.0, True, True)
    want = v[:, at].double().mean(1, keepdim=True)
    # the remainder's own rounding (h of at most h of the output), 1 / 3, the product and the three-term sum in fp32 (of terms up to the largest value)
    tol = h * h * want.abs() + 4 * 2.0 ** -24 * v[:, at].double().abs().amax(1, keepdim=True)
    assert ((out.double() + lo.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nk,d,q_block", [(16, 64, 64), (100, 128, 64), (1000, 64, 64), (700, 64, 1)])
@pytest.mark.parametrize("kind", ["mean 5", "mean 50", "no negative ones", "large scores"])
def test_gradients_of_values_with_a_common_part(kind, nk, d, q_block, dtype):
    """Values (and cotangents) of one sign or with a mean, and rows with one key of nearly all weight: rowsum(dout o out) and dout v^T are large and nearly the same.  The
    forward's roundings of the probabilities come into their difference by the values' distances from the output alone, that of what is kept of
    the output by h^2 of it."""
    g = torch.Generator().manual_seed(nk + d)
    nq, h = 256, half(dtype)
    size = 30.0 if kind == "large scores" else 1.5
    q, k, v, do = rnd(g, nq, d, scale=size), rnd(g, nk, d), rnd(g, nk, d), rnd(g, nq, d)
    if kind.startswith("mean"):
        v = v + float(kind[5:])
    if kind == "no negative ones":
        v, do = v.relu(), do.abs()
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    dq, dk, _ = gradients(q, k, v, do, q_block)
    Q, K, V, G = (t.to(DEV).double() for t in (q, k, v, do))
    c = d ** -0.5
    p, t, ds = dense(Q, K, V, G, c)
    delta = (p * t).square().sum(-1, keepdim=True) + h * h * (G * (p @ V)).square().sum(-1, keepdim=True)     # variance over h^2 / 3
    delta = delta * c * c
    for name, got, want, var in (("dq", dq, ds @ K, delta * (p @ K).square()), ("dk", dk, ds.T @ Q, (p * p * delta).T @ Q.square())):
        own = own_rounding(want, dtype)
        bound, err = 1.1 * (own ** 2 + h * h / 3 * var.sum().item()) ** 0.5, (got - want).norm().item()
        assert err <= bound, "%s: %.2f times its own rounding, bound %.2f" % (name, err / own, bound / own)
