"""GPU: the token lookup, preference loss, gradient clipping and 4-bit index operators against plain 64-bit
implementations, at the sizes, types, strides and masks where they can go wrong.

Tolerances count roundings: u = 2^-24 is half a step of fp32, HALF[t] half a step of the stored type.  A sum of m
fp32 terms is off by at most m u times the sum of their magnitudes; a stored value by HALF[t] of itself
(or half the smallest subnormal)."""
import math

import pytest
import torch

import twotower_amd as tt
from twotower_amd import _lib, losses, ops, optim

from test_operators_cpu import pair_terms

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}  # smallest subnormals


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check(got, want, bound, what=""):
    """|got - want| <= bound elementwise, finite and non-finite places alike."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    same = (got == want) | (got.isnan() & want.isnan())
    bad &= ~same
    if bad.any():
        i = bad.flatten().nonzero()[0].item()
        b = bound if not isinstance(bound, torch.Tensor) else bound.expand_as(want).flatten()[i].item()
        raise AssertionError(f"{what}: {bad.sum().item()} of {bad.numel()} off; first at {i}: got "
                             f"{got.flatten()[i].item()!r}, want {want.flatten()[i].item()!r}, bound {b}")


def stored(want, t):
    """How far a value of type t may be from `want` by its one rounding."""
    return want.abs() * HALF[t] + TINY[t]


# ---------------------------------------------------------------------------------------------
# token lookup
def lookup_case(V, E, shape, dtype, ids_dtype, out_dtype, pad, hot, seed):
    g = gen(seed)
    w = torch.randn(V, E, generator=g, device=DEV).to(dtype)
    ids = torch.randint(0, V, shape, generator=g, device=DEV)
    if hot:  # most tokens name one row
        ids = torch.where(torch.rand(shape, generator=g, device=DEV) < hot, torch.full_like(ids, V // 2), ids)
    if pad is not None:
        ids = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.4, torch.full_like(ids, pad % V), ids)
    dout = torch.randn(*shape, E, generator=g, device=DEV).to(out_dtype or dtype)
    return w, ids.to(ids_dtype), dout


def check_lookup(w, ids, dout, scale, pad, out_dtype, out, grad):
    V, E = w.shape
    flat = ids.reshape(-1).long()
    inside = (flat >= 0) & (flat < V)
    rows = w.double()[flat.clamp(0, V - 1)] * scale
    rows[~inside] = 0
    rows = rows.view(*ids.shape, E)
    t = out_dtype or w.dtype
    check(out, rows, 2 * U * rows.abs() + stored(rows, t), "rows")  # the factor and the product, then the type
    keep = inside & (flat != (pad % V if pad is not None else -1))
    d = dout.double().reshape(-1, E)[keep] * scale
    want = torch.zeros(V, E, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], d)
    mass = torch.zeros(V, E, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], d.abs())
    count = torch.zeros(V, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], torch.ones_like(d[:, 0]))
    check(grad, want, (count + 3).unsqueeze(1) * U * mass + stored(want, w.dtype), "gradient")
    assert not grad[count == 0].any()


LOOKUPS = [
    # V, E, ids shape, type, id type, out type, padding id, share of one hot row
    (34, 64, (64, 64), F32, torch.int64, None, 0, 0.0),          # 4096 tokens: the longest call without a sort
    (34, 64, (4097,), F32, torch.int64, None, 0, 0.0),           # one more
    (50_000, 128, (1, 64), BF16, torch.int32, None, 0, 0.0),
    (1, 1, (1,), F32, torch.int64, None, None, 0.0),
    (1, 5, (7000,), F16, torch.int32, None, None, 0.0),          # one row, every token its own
    (7, 1, (3, 5), BF16, torch.int64, None, -1, 0.0),            # padding id from the end
    (301, 100, (37, 29), F16, torch.int32, None, None, 0.0),
    (301, 100, (61, 83), F16, torch.int64, BF16, 3, 0.0),        # (refused: see below)
    (301, 100, (61, 83), F32, torch.int64, BF16, 3, 0.0),
    (301, 36, (61, 83), F32, torch.int32, F16, None, 0.0),
    (1000, 256, (4000,), F32, torch.int64, None, None, 0.9),     # a hot row shared by a workgroup
    (1000, 256, (60_000,), F32, torch.int64, None, None, 0.9),   # a hot row in pieces
    (129, 513, (5000,), F32, torch.int32, None, 1, 0.3),         # wider than a wave's accesses, odd
    (129, 1030, (300,), BF16, torch.int32, None, 1, 0.3),
    (70_000, 8, (20_000,), BF16, torch.int64, None, 0, 0.1),
    (2048, 512, (9000,), F16, torch.int64, None, 0, 0.5),
    (129, 513, (9000,), F32, torch.int32, None, 1, 0.3),
    (50, 65, (8192,), BF16, torch.int64, None, 0, 0.2),          # the longest call without a sort, and one more
    (50, 64, (8193,), BF16, torch.int64, None, 0, 0.2),
    (30, 600, (2000,), F32, torch.int32, None, None, 0.4),       # frequent rows of 3, 9 and 1 column chunks
    (40, 1030, (700,), F32, torch.int64, None, None, 0.5),
    (20, 1, (3000,), F32, torch.int64, None, None, 0.6),
    (20, 7, (257,), BF16, torch.int32, None, None, 1.0),         # one id alone
    (700, 256, (70_001,), F32, torch.int32, None, 0, 0.1),       # workgroups dealt to the XCDs in runs
]


@pytest.mark.parametrize("V, E, shape, dtype, ids_dtype, out_dtype, pad, hot", LOOKUPS)
def test_lookup_against_plain(V, E, shape, dtype, ids_dtype, out_dtype, pad, hot):
    w, ids, dout = lookup_case(V, E, shape, dtype, ids_dtype, out_dtype, pad, hot, 1)
    w.requires_grad_(True)
    if out_dtype is not None and dtype != F32:
        with pytest.raises(TypeError, match="out_dtype"):
            ops.embedding_lookup(w, ids, out_dtype=out_dtype)
        return
    scale = math.sqrt(E)
    out = ops.embedding_lookup(w, ids, scale=scale, padding_idx=pad, out_dtype=out_dtype)
    (grad,) = torch.autograd.grad(out, w, dout)
    assert out.dtype == (out_dtype or dtype) and grad.dtype == dtype
    check_lookup(w.detach(), ids, dout, scale, pad, out_dtype, out.detach(), grad)
    again = ops.embedding_lookup(w, ids, scale=scale, padding_idx=pad, out_dtype=out_dtype)
    assert torch.equal(torch.autograd.grad(again, w, dout)[0], grad)  # a fixed order: the same bits
    with torch.no_grad():
        assert torch.equal(ops.embedding_lookup(w, ids, scale=scale, out_dtype=out_dtype), out)


@pytest.mark.parametrize("n", [0, 600, 5000, 9000])
def test_lookup_ids_outside_the_table(n):
    V, E = 40, 24
    w, ids, dout = lookup_case(V, E, (n,), F32, torch.int64, None, None, 0.0, 2)
    ids[::3] = torch.tensor([-1, V, 2 ** 40, -2 ** 40], device=DEV).repeat(n)[:ids[::3].numel()]
    w.requires_grad_(True)
    out = ops.embedding_lookup(w, ids, scale=0.5)
    (grad,) = torch.autograd.grad(out, w, dout)
    check_lookup(w.detach(), ids, dout, 0.5, None, None, out.detach(), grad)


@pytest.mark.parametrize("n", [900, 9000])
def test_lookup_strides_and_alignment(n):
    g = gen(3)
    wide = torch.randn(500, 3 + 64 + 5, generator=g, device=DEV)
    ids = torch.randint(0, 500, (n // 30, 30), generator=g, device=DEV).t()  # not contiguous
    dout = torch.randn(30, n // 30, 64, generator=g, device=DEV).transpose(0, 1).contiguous().transpose(0, 1)
    for first in (0, 1, 2, 3):  # the rows start off a 16-byte boundary, their stride is wider than E
        w = wide[:, first:first + 64].detach().requires_grad_(True)
        out = ops.embedding_lookup(w, ids, scale=3.0, padding_idx=7)
        (grad,) = torch.autograd.grad(out, w, dout)
        check_lookup(w.detach(), ids, dout, 3.0, 7, None, out.detach(), grad)


@pytest.mark.parametrize("n", [900, 9000])
def test_lookup_non_finite_rows_stay_in_their_places(n):
    w, ids, dout = lookup_case(50, 16, (n,), F32, torch.int64, None, 0, 0.0, 4)
    w[0] = math.nan  # the padding row
    w[1] = math.inf
    dout[ids == 0] = math.nan  # gradients at padding tokens
    w.requires_grad_(True)
    out = ops.embedding_lookup(w, ids, scale=2.0, padding_idx=0)
    (grad,) = torch.autograd.grad(out, w, dout)
    assert torch.equal(out.isnan().all(-1), ids == 0) and torch.equal(out.isinf().all(-1), ids == 1)
    assert grad.isfinite().all() and not grad[0].any()


def test_lookup_odd_tables_and_ids():
    w = torch.arange(4.0, device=DEV)
    one = w.as_strided((1, 4), (1, 1)).detach().requires_grad_(True)  # one row: its stride says nothing
    col = torch.arange(12.0, device=DEV).view(6, 2)[:, :1].detach().requires_grad_(True)  # rows of one element
    for t in (one, col):
        out = ops.embedding_lookup(t, torch.tensor(0, device=DEV), scale=2.0)  # a scalar id
        assert torch.equal(out, 2.0 * t[0])
        (g,) = torch.autograd.grad(out.sum(), t)
        assert (g[0] == 2.0).all() and not g[1:].any()
    plain = torch.randn(9, 4, device=DEV, requires_grad=True)
    out = ops.embedding_lookup(plain * 3.0, torch.tensor([[1, 1]], device=DEV, dtype=torch.int32))  # not a leaf
    (g,) = torch.autograd.grad(out.sum(), plain)
    assert (g[1] == 6.0).all() and g.abs().sum() == 24.0
    with pytest.raises(RuntimeError, match="no second derivative"):  # said, not dropped
        torch.autograd.grad(losses.preference_loss(plain, plain.flip(0), plain.roll(1, 0)), plain, create_graph=True)


@pytest.mark.parametrize("n", [30, 6000, 9000])
@pytest.mark.parametrize("pad", [None, 2])
def test_lookup_differentiated_twice(n, pad):
    V, E = 12, 8  # small whole numbers: every sum is exact
    g = gen(12)
    w, c = (torch.randint(-3, 4, (V, E), generator=g, device=DEV).float() for _ in range(2))
    ids = torch.randint(-1, V, (n,), generator=g, device=DEV)
    x = torch.randint(-3, 4, (n, E), generator=g, device=DEV).float().requires_grad_(True)
    w.requires_grad_(True)
    out = ops.embedding_lookup(w, ids, scale=2.0, padding_idx=pad)
    (dw,) = torch.autograd.grad((out * out * x).sum(), w, create_graph=True)  # 8 w sum of x, each row's
    d2w, dx = torch.autograd.grad((dw * c).sum(), (w, x))
    keep = (ids >= 0) & (ids != (-9 if pad is None else pad))
    sums = torch.zeros(V, E, device=DEV).index_add_(0, ids[keep], x.detach()[keep])
    assert torch.equal(dw.detach(), 8 * w.detach() * sums) and torch.equal(d2w, 8 * c * sums)
    assert torch.equal(dx, torch.where(keep[:, None], 8 * (w.detach() * c)[ids], torch.zeros((), device=DEV)))


@pytest.mark.parametrize("dtype, out_dtype", [(F32, None), (F32, BF16), (F16, None)])
@pytest.mark.parametrize("leaf", [False, True])
def test_lookup_of_a_dual_table(leaf, dtype, out_dtype):
    """Forward mode: the rows' tangents are the tangent's rows, whether or not the table needs a gradient too."""
    from torch.autograd import forward_ad

    w, ids, _ = lookup_case(40, 24, (5, 9), dtype, torch.int64, out_dtype, 0, 0.0, 14)
    ids[0, 0] = 40  # outside
    t = torch.randn(24, 40, generator=gen(14), device=DEV).to(dtype).t()  # its own layout
    w.requires_grad_(leaf)
    with forward_ad.dual_level():
        plain = ops.embedding_lookup(w, ids, 4.0, 0, out_dtype)  # no tangent
        assert forward_ad.unpack_dual(plain).tangent is None
        out = ops.embedding_lookup(forward_ad.make_dual(w, t), ids, 4.0, 0, out_dtype)
        rows, tangent = forward_ad.unpack_dual(out)
        assert torch.equal(rows, plain) and rows.requires_grad == leaf
        assert torch.equal(tangent, ops.embedding_lookup(t.contiguous(), ids, 4.0, None, out_dtype))
        if leaf:
            d = torch.randn(rows.shape, generator=gen(15), device=DEV).to(rows.dtype)
            assert torch.equal(*(torch.autograd.grad(x, w, d)[0] for x in (rows, plain)))
    with pytest.raises(RuntimeError):  # a function transform's tensors have no memory of their own
        torch.func.jvp(lambda x: ops.embedding_lookup(x, ids, 4.0, 0, out_dtype), (w.detach(),), (t.contiguous(),))


def test_lookup_of_a_fused_table():
    """The fused update takes pooled lookups: a step that also differentiates a plain one is refused, a step with
    plain ones alone takes the dense gradient as any parameter does."""
    emb = tt.embeddings.build("lookup", vocab_size=30, embedding_dim=64).to(DEV)
    opt = optim.AdamW(emb.parameters(), fused_tables=True, tables=[emb])
    ids = torch.randint(1, 30, (3, 5), generator=gen(11), device=DEV)
    before = emb.weight.detach().clone()
    emb(ids).sum().backward()
    opt.step()
    assert not torch.equal(emb.weight, before)
    opt.zero_grad(set_to_none=True)
    (emb(ids).sum() + emb.pool_mean(ids).sum()).backward()
    with pytest.raises(RuntimeError, match="pooled lookups only"):
        opt.step()
    opt.zero_grad(set_to_none=True)
    emb.pool_mean(ids).sum().backward()
    opt.step()


def test_lookup_backward_through_a_loss_matches_differences():
    w, ids, _ = lookup_case(9, 6, (4, 5), F32, torch.int64, None, 0, 0.0, 5)
    ids[0, :2] = 3  # the same id twice
    w.requires_grad_(True)
    (grad,) = torch.autograd.grad((ops.embedding_lookup(w, ids, scale=1.5, padding_idx=0) ** 2).sum(), w)

    def f(x):  # the loss in 64 bits
        return ((x[ids] * 1.5) ** 2).sum()

    x, step = w.detach().double(), 1e-4
    for r in range(1, 9):
        for e in range(6):
            lo, hi = x.clone(), x.clone()
            lo[r, e] -= step
            hi[r, e] += step
            want = (f(hi) - f(lo)).item() / (2 * step)  # (exact for a square, up to 2^-53 f / step < 1e-10)
            assert abs(grad[r, e].item() - want) <= 30 * U * abs(want) + 1e-9


@pytest.mark.parametrize("n", [700, 8000, 30_000])
def test_lookup_captured_and_replayed(n):
    V, E = 400, 64
    w, ids, dout = lookup_case(V, E, (n,), F32, torch.int64, None, 0, 0.2, 6)
    w.requires_grad_(True)

    def step():
        out = ops.embedding_lookup(w, ids, scale=2.0, padding_idx=0)
        return out.detach(), torch.autograd.grad(out, w, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        ids.copy_(torch.randint(0, V, (n,), generator=gen(60 + k), device=DEV))
        dout.copy_(torch.randn(n, E, generator=gen(70 + k), device=DEV))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k


def test_lookup_on_another_stream():
    w, ids, dout = lookup_case(3000, 64, (20_000,), F32, torch.int64, None, 0, 0.1, 7)
    w.requires_grad_(True)
    want = torch.autograd.grad(ops.embedding_lookup(w, ids), w, dout)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(ops.embedding_lookup(w, ids), w, dout)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_lookup_offsets_beyond_32_bits():
    V, E, n = 1000, 512, 4_300_000  # 2.2e9 output elements
    w = torch.randn(V, E, generator=gen(8), device=DEV).to(BF16).requires_grad_(True)
    ids = torch.randint(0, V, (n,), generator=gen(9), device=DEV, dtype=torch.int32)
    out = ops.embedding_lookup(w, ids)
    assert torch.equal(out[-3:], w[ids[-3:].long()])
    ids.clamp_(0, V - 2)
    ids[-2:] = V - 1
    dout = torch.zeros_like(out)
    dout[-2:] = 1.0
    (grad,) = torch.autograd.grad(ops.embedding_lookup(w, ids), w, dout)
    assert (grad[-1] == 2.0).all() and not grad[:-1].any()


@pytest.mark.parametrize("V, n", [(140_000_001, 90), (300_000_001, 9000)])
def test_lookup_gradient_of_a_very_long_table(V, n):
    """More workgroups than one grid dimension takes (short and long calls)."""
    w = torch.zeros(V, 1, dtype=F16, device=DEV, requires_grad=True)
    ids = V - 1 - torch.arange(n, device=DEV) // 3
    ids[:2] = torch.tensor([0, V // 2], device=DEV)
    (grad,) = torch.autograd.grad(ops.embedding_lookup(w, ids, scale=0.5).sum(), w)
    want = torch.zeros(V, 1, device=DEV).index_add_(0, ids, torch.full((n, 1), 0.5, device=DEV))
    assert torch.equal(grad.float(), want)


def test_rows_beyond_one_grid_dimension():
    n = 33_600_005
    ids = torch.arange(n, device=DEV, dtype=torch.int32) % 37
    w = torch.randn(37, 65, generator=gen(14), device=DEV).to(F16)
    out = ops.embedding_lookup(w, ids)
    for lo in (0, n // 2, n - 100_000):
        assert torch.equal(out[lo:lo + 100_000], w[ids[lo:lo + 100_000].long()])
    del out
    B = 8_400_003  # whole numbers: every sum and gradient is exact
    q, p, nn = (torch.randint(-1, 2, (B, 65), generator=gen(15 + i), device=DEV).to(BF16).requires_grad_(True) for i in range(3))
    assert torch.equal(losses.preference_margin(q, p, nn, 1.0), (q * (p - nn)).float().sum(1, keepdim=True))
    loss = losses.preference_loss(q, p, nn, beta=0.5, temperature=1.0, loss_type="squared")
    dq, _, dn = torch.autograd.grad(loss, (q, p, nn), torch.tensor(float(B), device=DEV))
    with torch.no_grad():
        c = 2 * ((q * (p - nn)).float().sum(1, keepdim=True) - 1)
        for got, want in ((dq, c * (p - nn)), (dn, -c * q)):  # B (1 / B) is off by 2 U, then the rounding to bf16
            assert ((got - want).abs() <= (2 ** -8 + 4 * U) * want.abs()).all()
    del q, p, nn, dq, dn, c, got, want
    rows = ops.Int4Rows.quantize(torch.randint(-7, 8, (n, 8), generator=gen(19), device=DEV, dtype=torch.int8).to(BF16))
    x = rows.dequantize()
    g = torch.randint(-7, 8, (n, 8), generator=gen(19), device=DEV, dtype=torch.int8).float()
    full = g.abs().amax(1, keepdim=True) == 7  # scale 1: the codes are the values
    assert torch.equal(torch.where(full, x, g), g)


def test_lookup_embedding_module_uses_the_kernels():
    emb = tt.embeddings.build("lookup", vocab_size=50, embedding_dim=16, scale=4.0).to(DEV)
    ids = torch.randint(0, 50, (3, 7), generator=gen(10), device=DEV)
    with _lib.record_calls() as calls:
        out = emb(ids)
        out.sum().backward()
    assert {"tt_lookup_fwd", "tt_lookup_bwd"} <= calls
    assert torch.equal(out, emb.embedding(ids) * 4.0)  # a power of two: no rounding
    count = torch.zeros(50, device=DEV).index_add_(0, ids.flatten(), torch.ones(21, device=DEV))
    count[0] = 0  # the padding row
    assert torch.equal(emb.embedding.weight.grad, (4.0 * count).unsqueeze(1).expand(50, 16))


def test_calls_are_timed_and_recorded_on_autograds_thread():
    w = torch.randn(50, 16, device=DEV, requires_grad=True)
    q, p, n = (torch.randn(4, 16, device=DEV, requires_grad=True) for _ in range(3))
    _lib.TIMER.reset()
    _lib.TIMER.enabled = True
    try:
        ops.embedding_lookup(w, torch.arange(9, device=DEV)).sum().backward()
        losses.preference_loss(q, p, n).backward()
        optim.clip_grad_norm_([w, q, p, n], 1.0)
    finally:
        _lib.TIMER.enabled = False
    got = _lib.TIMER.summary()
    _lib.TIMER.reset()
    names = {"tt_lookup_fwd", "tt_lookup_bwd", "tt_preference_fwd", "tt_preference_bwd", "tt_clip_grads"}
    assert names <= set(got) and all(got[k]["calls"] == 1 and got[k]["total_ms"] > 0 for k in names)


def test_lookups_of_two_threads_at_once():
    import threading

    cases = [lookup_case(3000, 64, (n,), F32, torch.int64, None, 0, 0.1, 15 + n) for n in (700, 20_000)]
    for w, _, _ in cases:
        w.requires_grad_(True)

    def grad(w, ids, dout):
        return torch.autograd.grad(ops.embedding_lookup(w, ids, 2.0, 0), w, dout)[0]

    want = [grad(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got[i] = [grad(*cases[i]) for _ in range(20)]
        side.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(g) == 20 and all(torch.equal(x, want[i]) for x in g) for i, g in enumerate(got))


def test_lookup_embedding_module_under_torchs_transforms():
    """What follows torch's own calls (function transforms, tracing, dispatch modes, hooks) sees the plain gather."""
    emb = tt.embeddings.build("lookup", vocab_size=50, embedding_dim=16, scale=4.0).to(DEV)
    ids = torch.randint(0, 50, (3, 7), generator=gen(13), device=DEV)
    w = emb.embedding.weight.detach()

    def f(x):
        return torch.func.functional_call(emb, {"embedding.weight": x}, (ids,)).square().sum()

    x = w.clone().requires_grad_(True)
    want = torch.autograd.grad(f(x), x)[0]  # the kernels: rows times a power of two, few terms a row
    assert (torch.func.grad(f)(w) - want).abs().max() <= 32 * U * want.abs().max()  # (at most 21 terms a sum)
    _, tangent = torch.func.jvp(f, (w,), (torch.ones_like(w),))
    rows = emb.embedding(ids).detach()
    assert abs(tangent.item() - 32 * rows.double().sum().item()) <= 32 * 336 * U * rows.abs().sum().item()
    with torch.no_grad():
        traced = torch.jit.trace(emb, (ids,))
        with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True):
            assert emb(torch.empty(2, 5, dtype=torch.int64, device=DEV)).shape == (2, 5, 16)
        other = (ids + 1) % 50
        assert torch.equal(traced(other), emb(other))
    seen = []
    hook = emb.embedding.register_forward_hook(lambda *a: seen.append(1))
    emb(ids)
    hook.remove()
    assert seen == [1]


@pytest.mark.parametrize("how", [torch.fx.symbolic_trace, torch.jit.script, lambda m: torch.compile(m, backend="eager", fullgraph=True)],
                         ids=["fx", "script", "compile"])
def test_lookup_embedding_module_traced_and_compiled(how):
    emb = tt.embeddings.build("lookup", vocab_size=50, embedding_dim=16, scale=4.0).to(DEV)
    ids = torch.randint(0, 50, (3, 7), generator=gen(17), device=DEV)
    got, want = how(emb)(ids), emb(ids)
    assert torch.equal(got, want)
    a, b = (torch.autograd.grad(x.square().sum(), emb.weight)[0] for x in (got, want))
    assert (a - b).abs().max() <= 32 * U * b.abs().max()  # (at most 21 terms a sum)


@pytest.mark.parametrize("dtype, out_dtype", [(F32, None), (BF16, None), (F16, None), (F32, F16)])
@pytest.mark.parametrize("n", [5, 900, 70_000])
def test_strict_lookup_of_ids_outside_the_table(n, dtype, out_dtype):
    w, ids, dout = lookup_case(700, 64, (n,), dtype, torch.int64, out_dtype, 0, 0.0, 18)
    ids[::5] = torch.tensor([700, -1, 2 ** 40, -2 ** 63], device=DEV).repeat(n)[:len(ids[::5])]
    out = (ids < 0) | (ids >= 700)
    w.requires_grad_(True)
    got = ops.embedding_lookup(w, ids, 3.0, 0, out_dtype, strict=True)
    loose = ops.embedding_lookup(w, ids, 3.0, 0, out_dtype)
    assert got[out].isnan().all() and torch.equal(got[~out], loose[~out]) and not loose[out].any()
    assert torch.equal(*(torch.autograd.grad(x, w, dout)[0] for x in (got, loose)))


def test_a_wrong_vocabulary_does_not_train_silently():
    emb = tt.embeddings.build("lookup", vocab_size=50, embedding_dim=16, scale=4.0).to(DEV)
    ids = torch.randint(0, 50, (3, 7), generator=gen(19), device=DEV)
    fine = emb(ids)
    assert fine.isfinite().all()
    ids[1, 2] = 50
    rows = emb(ids)
    assert rows[1, 2].isnan().all() and rows.isnan().sum() == 16
    assert rows.square().mean().isnan()
    rows.logsumexp((0, 1, 2)).backward()  # (a loss that joins its tokens; the squares' other terms stay finite)
    assert emb.weight.grad.isnan().any() and optim.clip_grad_norm_(emb.parameters(), 1.0).isnan()
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(emb.weight.detach(), torch.ones_like(emb.weight))
        rows = torch.autograd.forward_ad.unpack_dual(ops.embedding_lookup(t, ids, strict=True))
        assert rows.primal[1, 2].isnan().all() and not rows.tangent[1, 2].any()


def test_lookup_embedding_module_runs_what_is_around_the_inner_one():
    """Global hooks, a forward of the instance's own and function modes see torch's gather; a default device does not
    turn the kernels off."""
    emb = tt.embeddings.build("lookup", vocab_size=50, embedding_dim=16, scale=4.0).to(DEV)
    ids = torch.randint(0, 50, (3, 7), generator=gen(16), device=DEV)
    want = emb(ids)
    seen = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: seen.append(type(m)))
    try:
        assert torch.equal(emb(ids), want)
    finally:
        handle.remove()
    assert torch.nn.Embedding in seen
    plain = emb.embedding.forward
    emb.embedding.forward = lambda x: plain(x) + 1.0
    assert torch.equal(emb(ids), (emb.weight[ids] + 1.0) * 4.0)
    del emb.embedding.forward
    names = []

    class Mode(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            names.append(getattr(func, "__name__", ""))
            return func(*args, **(kwargs or {}))

    with Mode():
        assert torch.equal(emb(ids), want)
    assert "embedding" in names
    with torch.device("cpu"), _lib.record_calls() as calls:
        assert torch.equal(emb(ids), want)
    assert "tt_lookup_fwd" in calls


# ---------------------------------------------------------------------------------------------
# preference loss
def pref_case(B, H, K, dtype, ref, mask, seed):
    g = gen(seed)

    def rows(*shape):
        return torch.nn.functional.normalize(torch.randn(*shape, H, generator=g, device=DEV), dim=-1).to(dtype)

    q, p, n = rows(B), rows(B), rows(B, K)
    r = torch.randn(B, K, generator=g, device=DEV) + 1.0 if ref else None
    m = torch.rand(B, K, generator=g, device=DEV) >= mask if mask else None
    return q, p, n, r, m


def check_pref(q, p, n, r, m, got, beta=0.5, temperature=0.1, smooth=0.0, kind="sigmoid", upstream=1.0):
    """got = (loss, dq, dp, dn) against the formulas in 64 bits, within the roundings of an fp32 evaluation."""
    B, K, H = n.shape
    on = torch.ones(B, K, dtype=torch.bool, device=DEV) if m is None else m
    any_on = on.any(1)
    # absent rows count as zeros: nothing of them may reach a result
    Q = torch.where(any_on.unsqueeze(1), q.double(), 0.0)
    P = torch.where(any_on.unsqueeze(1), p.double(), 0.0)
    N = torch.where(on.unsqueeze(2), n.double(), 0.0)
    D = (P.unsqueeze(1) - N) * on.unsqueeze(2)
    h = (Q.unsqueeze(1) * D).sum(2) / temperature - (0 if r is None else r.double())
    l, dl = pair_terms(h, beta, smooth, kind)
    l, dl = l * on, dl * on
    pairs = max(1, int(on.sum()))
    # h: difference, H products and sums, 1 / temperature and its product, the subtraction of ref
    eh = ((H + 5) * U * (Q.unsqueeze(1) * D).abs().sum(2) / temperature + 2 * U * (h.abs() + (0 if r is None else r.double().abs()))) * on
    if kind == "sigmoid":  # |l'| <= beta; l'' <= beta^2 / 4; exp and log1p within 4 steps, sigma and the sums a few more
        el = beta * eh + 16 * U * (l + on * math.log(2))
        ed = beta ** 2 / 4 * eh + 16 * U * beta * on
        ed = ed + beta * 4 * U * (beta * h).abs() * torch.exp(-(beta * h).abs())  # the rounding of beta h
    else:
        el = 2 * (h - 0.5 / beta).abs() * (eh + 4 * U * (h.abs() + 0.5 / beta)) + (eh + 4 * U * (h.abs() + 0.5 / beta)) ** 2 + 2 * U * l
        ed = 2 * (eh + 4 * U * (h.abs() + 0.5 / beta)) * on
    loss, dq, dp, dn = got
    check(loss, upstream ** 0 * l.sum() / pairs, el.sum() / pairs + (K + 4) * U * l.sum() / pairs, "loss")
    G = upstream / (pairs * temperature)
    wq = G * (dl.unsqueeze(2) * D).sum(1)
    bq = abs(G) * ((ed + (K + 6) * U * dl.abs()).unsqueeze(2) * D.abs()).sum(1)
    wp = G * dl.sum(1, keepdim=True) * Q
    bp = abs(G) * (ed + (K + 6) * U * dl.abs()).sum(1, keepdim=True) * Q.abs()
    wn = -G * dl.unsqueeze(2) * Q.unsqueeze(1)
    bn = abs(G) * (ed + 6 * U * dl.abs()).unsqueeze(2) * Q.unsqueeze(1).abs()
    for a, w, b, t, nm in ((dq, wq, bq, q, "dq"), (dp, wp, bp, p, "dp"), (dn, wn, bn, n, "dn")):
        check(a, w, b + stored(w.abs() + b, t.dtype), nm)


PREFS = [
    # B, H, K, type, ref, masked share, beta, temperature, smoothing, kind
    (64, 128, 1, F32, False, 0.0, 1.0, 0.1, 0.0, "sigmoid"),
    (8192, 256, 1, F32, True, 0.0, 0.5, 0.1, 0.1, "sigmoid"),
    (1000, 256, 4, BF16, True, 0.3, 0.5, 0.1, 0.0, "squared"),
    (1, 1, 1, F32, False, 0.0, 0.1, 0.1, 0.0, "sigmoid"),
    (3, 7, 5, F16, True, 0.5, 1.0, 0.05, 0.0, "sigmoid"),
    (257, 100, 2, BF16, False, 0.0, 0.1, 1.0, 0.3, "sigmoid"),
    (33, 1030, 9, F32, True, 0.8, 0.5, 0.1, 0.0, "squared"),
    (129, 2048, 1, BF16, False, 0.0, 1.0, 0.05, 0.0, "sigmoid"),
    (5000, 20, 3, F16, True, 0.9, 1.0, 0.1, 0.0, "squared"),
    (33, 382, 8, F16, True, 0.0, 0.1, 0.05, 0.0, "squared"),       # columns side by side in the backward
    (2, 5001, 5, F32, False, 0.0, 0.5, 0.1, 0.1, "sigmoid"),
    (40, 1, 9, BF16, True, 0.4, 0.5, 0.1, 0.0, "sigmoid"),         # one lane a query, several rounds of pairs
    (40, 2, 6, F32, True, 0.4, 0.5, 0.1, 0.2, "sigmoid"),
    (16, 256, 4, F32, False, 0.2, 1.0, 0.1, 0.0, "sigmoid"),       # one workgroup, four pairs together
    (128, 128, 8, BF16, True, 0.2, 1.0, 0.1, 0.0, "squared"),
]


@pytest.mark.parametrize("B, H, K, dtype, ref, mask, beta, temperature, smooth, kind", PREFS)
def test_preference_against_plain(B, H, K, dtype, ref, mask, beta, temperature, smooth, kind):
    q, p, n, r, m = pref_case(B, H, K, dtype, ref, mask, 20)
    for t in (q, p, n):
        t.requires_grad_(True)
    kw = dict(beta=beta, temperature=temperature, label_smoothing=smooth, loss_type=kind)
    loss = losses.preference_loss(q, p, n, ref_margin=r, mask=m, **kw)
    assert loss.dtype == F32 and loss.dim() == 0
    grads = torch.autograd.grad(loss, (q, p, n))
    check_pref(q.detach(), p.detach(), n.detach(), r, m, (loss.detach(), *grads), beta, temperature, smooth, kind)
    again = losses.preference_loss(q, p, n, ref_margin=r, mask=m, **kw)
    assert torch.equal(again, loss)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, (q, p, n)), grads))


def test_preference_masked_pairs_are_not_read():
    q, p, n, r, _ = pref_case(40, 64, 3, F32, True, 0.0, 21)
    m = torch.ones(40, 3, dtype=torch.bool, device=DEV)
    m[::4, 1] = False
    m[5] = False  # a query with no pair left
    n[~m] = math.nan
    r[~m] = math.inf
    q[5], p[5] = math.nan, math.inf
    for t in (q, p, n):
        t.requires_grad_(True)
    loss = losses.preference_loss(q, p, n, ref_margin=r, mask=m, beta=0.5)
    grads = torch.autograd.grad(loss, (q, p, n))
    assert not grads[0][5].any() and not grads[1][5].any() and not grads[2][~m].any()
    check_pref(q.detach(), p.detach(), n.detach(), torch.where(m, r, 0.0), m, (loss.detach(), *grads))


@pytest.mark.parametrize("B", [0, 1, 700, 30_000])
def test_preference_with_no_pair(B):
    q, p, n, _, _ = pref_case(B, 16, 2, F32, False, 0.0, 22)
    m = torch.zeros(B, 2, dtype=torch.bool, device=DEV)
    for t in (q, p, n):
        t.requires_grad_(True)
    loss = losses.preference_loss(q, p, n, mask=m)
    assert loss.item() == 0.0
    assert all(not g.any() and g.shape == t.shape for g, t in zip(torch.autograd.grad(loss, (q, p, n)), (q, p, n)))


def test_preference_extreme_margins():
    q = torch.ones(4, 1, device=DEV, requires_grad=True)
    p = torch.tensor([[1e4], [-1e4], [100.0], [-100.0]], device=DEV, requires_grad=True)
    n = torch.zeros(4, 1, device=DEV, requires_grad=True)
    loss = losses.preference_loss(q, p, n, beta=1.0, temperature=1.0)
    dq, dp, dn = torch.autograd.grad(loss, (q, p, n))
    # softplus(-h): 0, 1e4, e^-100 (below 2^-126), 100; its derivative -sigma(-h): 0, -1, ~0, -1
    assert abs(loss.item() - 10100 / 4) <= 4 * U * 10100
    want = torch.tensor([[0.0], [-0.25], [0.0], [-0.25]], dtype=torch.float64, device=DEV)
    check(dp, want, 1e-40 + U, "dp")
    check(dn, -want, 1e-40 + U, "dn")
    assert dq.isfinite().all()
    (g,) = torch.autograd.grad(losses.preference_loss(q, p, n, beta=1.0, temperature=1.0) * 3.0, p)
    check(g, 3 * want, 4 * U, "upstream")


def test_preference_strides():
    g = gen(23)
    wide = torch.randn(50, 5 + 96, generator=g, device=DEV)
    negs = torch.randn(3, 50, 100, generator=g, device=DEV)  # (K, B, H + 4)
    q, p = wide[:, 5:37], wide[:, 64:96]
    n = negs.permute(1, 0, 2)[:, :, 2:34]
    odd = torch.randn(50, 32, 2, generator=g, device=DEV)[..., 0]  # elements two apart
    for a, b, c in ((q, p, n), (odd, p, n), (q, odd, negs.permute(1, 0, 2)[:, :, :32])):
        a, b, c = (t.detach().requires_grad_(True) for t in (a, b, c))
        loss = losses.preference_loss(a, b, c, beta=0.5, temperature=5.0)
        grads = torch.autograd.grad(loss, (a, b, c))
        check_pref(a.detach(), b.detach(), c.detach(), None, None, (loss.detach(), *grads), temperature=5.0)


@pytest.mark.parametrize("K", [1, 3])
def test_preference_on_the_fused_tower_output(K):
    B, H = 60, 64
    base = torch.randn((2 + K) * B, H, generator=gen(24), device=DEV, requires_grad=True)
    y = base * 0.3
    q, p, n = torch.split(y, [B, B, K * B])
    n3 = n if K == 1 else n.view(B, K, H)
    loss = losses.preference_loss(q, p, n3, beta=0.5)
    assert "Packed" in loss.grad_fn.name()
    (got,) = torch.autograd.grad(loss, base)
    a, b, c = (t.detach().clone().requires_grad_(True) for t in (q, p, n3))
    want = torch.autograd.grad(losses.preference_loss(a, b, c, beta=0.5), (a, b, c))
    assert torch.equal(got, torch.cat([t.reshape(-1, H) for t in want]) * 0.3)


def test_preference_on_views_that_are_their_own_leaves():
    x = torch.randn(60, 32, generator=gen(28), device=DEV)
    q, p, n = (t.requires_grad_(True) for t in x.split([20, 20, 20]))  # blocks of a tensor without a gradient
    loss = losses.preference_loss(q, p, n, beta=0.5)
    got = torch.autograd.grad(loss, (q, p, n))
    a, b, c = (t.detach().clone().requires_grad_(True) for t in (q, p, n))
    assert all(torch.equal(u, v) for u, v in zip(got, torch.autograd.grad(losses.preference_loss(a, b, c, beta=0.5), (a, b, c))))
    y = x.clone().requires_grad_(True)
    with torch.no_grad():
        q = y[:20]  # no gradient is wanted through the queries
    loss = losses.preference_loss(q, y[20:40], y[40:], beta=0.5)
    (g,) = torch.autograd.grad(loss, y)
    assert not g[:20].any() and torch.equal(g[20:40], got[1]) and torch.equal(g[40:], got[2])


class _Halved(torch.autograd.Function):
    """A view whose gradient is scaled (gradient scaling or reversal layers have this form)."""

    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        return g * 0.5


@pytest.mark.parametrize("split", [torch.split, ops.split_rows])
@pytest.mark.parametrize("K", [1, 3])
def test_preference_sees_what_autograd_has_on_the_blocks(K, split):
    """Blocks of one tensor: a function between a block and the loss, hooks, retained gradients, and gradients with
    respect to the blocks, against the same loss of separate tensors."""
    B, H = 37, 48
    x = torch.randn((2 + K) * B, H, generator=gen(29), device=DEV)

    def blocks():
        leaf = x.clone().requires_grad_(True)
        return leaf, list(split(leaf * 1.0, [B, B, K * B]))

    def loss(q, p, n):
        return losses.preference_loss(q, p, n if K == 1 else n.view(B, K, H), beta=0.5)

    alone = [t.clone().requires_grad_(True) for t in x.split([B, B, K * B])]
    want = torch.autograd.grad(loss(*alone), alone)
    leaf, parts = blocks()
    (got,) = torch.autograd.grad(loss(*parts), leaf)
    assert torch.equal(got, torch.cat(want))
    leaf, parts = blocks()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss(*parts), parts), want))
    for i in range(3):
        leaf, parts = blocks()
        out = loss(*[_Halved.apply(t) if j == i else t for j, t in enumerate(parts)])
        (got,) = torch.autograd.grad(out, leaf)
        assert torch.equal(got, torch.cat([w * (0.5 if j == i else 1.0) for j, w in enumerate(want)]))
        leaf, parts = blocks()
        seen = []
        parts[i].register_hook(lambda g: seen.append(g.clone()))
        parts[i].register_hook(lambda g: g * 4.0)
        parts[(i + 1) % 3].retain_grad()
        loss(*parts).backward()
        assert torch.equal(seen[0], want[i]) and torch.equal(parts[(i + 1) % 3].grad, want[(i + 1) % 3])
        assert torch.equal(leaf.grad, torch.cat([w * (4.0 if j == i else 1.0) for j, w in enumerate(want)]))


@pytest.mark.parametrize("name", ["triplet", "multiple_negatives", "in_batch"])
def test_contrastive_losses_see_what_autograd_has_on_the_blocks(name):
    B, H = 32, 64
    x = torch.randn(3 * B, H, generator=gen(31), device=DEV)
    fn = losses.build(name)

    def blocks():
        leaf = x.clone().requires_grad_(True)
        return leaf, list(torch.split(leaf * 1.0, B))

    alone = [t.clone().requires_grad_(True) for t in x.split(B)]
    want = torch.autograd.grad(fn(*alone), alone)

    def same(got, scale):  # (the two forms of a loss may differ by roundings)
        for j, w in enumerate(want):
            assert (got[j * B:(j + 1) * B] - scale[j] * w).norm() <= 1e-5 * w.norm()

    leaf, parts = blocks()
    same(torch.autograd.grad(fn(*parts), leaf)[0], (1, 1, 1))
    for split in (torch.split, lambda y, n: ops.split_rows(y, [n] * 3)):  # with respect to the blocks, and late hooks
        y = x.clone().requires_grad_(True) * 1.0
        parts = split(y, B)
        loss = fn(*parts)
        assert "Packed" in loss.grad_fn.name()
        same(torch.cat(torch.autograd.grad(loss, parts, retain_graph=True)), (1, 1, 1))
        parts[1].register_hook(lambda g: g * 2)
        same(torch.autograd.grad(loss, y)[0], (1, 2, 1))
    for i in range(3):
        scale = [0.5 if j == i else 1.0 for j in range(3)]
        leaf, parts = blocks()
        same(torch.autograd.grad(fn(*[_Halved.apply(t) if j == i else t for j, t in enumerate(parts)]), leaf)[0], scale)
        leaf, parts = blocks()
        parts[i].register_hook(lambda g: g * 0.5)
        same(torch.autograd.grad(fn(*parts), leaf)[0], scale)
        leaf, parts = blocks()
        parts[i].retain_grad()
        fn(*parts).backward()
        assert (parts[i].grad - want[i]).norm() <= 1e-5 * want[i].norm()


def test_preference_gradient_of_the_tower_output_is_not_copied():
    torch.manual_seed(30)
    emb = tt.embeddings.build("lookup", vocab_size=60, embedding_dim=64)
    model = tt.build_two_tower("mean", emb, hidden_dim=128, tied_weights=True).to(DEV)
    ids = torch.randint(1, 60, (3, 20, 8), generator=gen(30), device=DEV)
    q, p, n = model(*ids)
    base = q._base
    base.retain_grad()
    seen = []
    q.register_hook(lambda g: seen.append(g.data_ptr()))
    whole = []
    base.register_hook(lambda g: whole.append(g.data_ptr()))
    losses.preference_loss(q, p, n, beta=0.5).backward()
    assert seen == whole  # the loss's own buffer
    alone = [t.detach().requires_grad_(True) for t in (q, p, n)]
    assert torch.equal(base.grad, torch.cat(torch.autograd.grad(losses.preference_loss(*alone, beta=0.5), alone)))


def test_preference_margin_is_the_reference_term():
    q, p, n, _, _ = pref_case(77, 48, 2, BF16, False, 0.0, 25)
    r = losses.preference_margin(q.requires_grad_(True), p, n, temperature=0.1)
    assert not r.requires_grad and r.shape == (77, 2)
    loss = losses.preference_loss(q, p, n, ref_margin=r, beta=0.5, temperature=0.1)
    assert abs(loss.item() - math.log(2)) <= 8 * U  # the model is its own reference: every margin is 0
    one = losses.preference_loss(q, p, n[:, 0], ref_margin=r[:, 0], beta=0.5)
    assert abs(one.item() - math.log(2)) <= 8 * U


@pytest.mark.parametrize("B", [30, 3000])
def test_preference_captured_and_replayed(B):
    q, p, n, r, m = pref_case(B, 64, 2, F32, True, 0.3, 26)
    for t in (q, p, n):
        t.requires_grad_(True)

    def step():
        loss = losses.preference_loss(q, p, n, ref_margin=r, mask=m, beta=0.5)
        return (loss.detach(), *torch.autograd.grad(loss, (q, p, n)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        new = pref_case(B, 64, 2, F32, True, 0.3 if k < 2 else 1.1, 27 + k)
        with torch.no_grad():
            for old, t in zip((q, p, n, r, m), new):
                old.copy_(t)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


# ---------------------------------------------------------------------------------------------
# gradient norm and clipping
def clip_case(sizes, types, seed, scale=1.0):
    g = gen(seed)
    return [(torch.randn(s, generator=g, device=DEV) * scale).to(t) for s, t in zip(sizes, types)]


def check_clip(grads, outs, norm, max_norm, kind):
    every = torch.cat([x.double().flatten() for x in grads]) if grads else torch.zeros(1, device=DEV).double()
    want = every.abs().max() if kind == math.inf else every.square().sum().sqrt()
    check(norm, want, 1.001 * U * want, "norm")  # 64-bit sums of n terms: n 2^-53, then one fp32 rounding
    coef = (max_norm / (want + 1e-6)).clamp(max=1.0)
    for i, (g, o) in enumerate(zip(grads, outs)):
        w = g.double() * coef  # the factor's rounding, the product's, the type's
        check(o, w, 2.001 * U * w.abs() + stored(w, o.dtype), f"tensor {i}")


CLIPS = [
    ([65536, 256, 65536, 256], [F32] * 4, 1.0, 2.0),
    ([1], [F32], 0.5, 2.0),
    ([16384, 16385, 16383, 7], [BF16] * 4, 1.0, 2.0),
    ([5, 0, 70001, 3], [F16, F32, BF16, F32], 1.0, 2.0),
    ([5, 0, 70001, 3], [F16, F32, BF16, F32], 0.3, math.inf),
    ([100_003], [F32], 1e6, 2.0),   # not clipped
    ([1000] * 168, [F32] * 168, 1.0, 2.0),   # one launch, and one tensor more
    ([1000, 3] * 84 + [2049], [F32] * 169, 1.0, 2.0),
    ([97] * 129 + [30_000] * 150, [F32, BF16, F16] * 93, 1.0, 2.0),  # several launches
]


@pytest.mark.parametrize("sizes, types, max_norm, kind", CLIPS)
def test_clip_against_plain(sizes, types, max_norm, kind):
    grads = clip_case(sizes, types, 30)
    before = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, None, norm_type=kind)  # the norm alone changes nothing
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    outs = list(torch.split(torch.full((sum(sizes),), 7.0, device=DEV), sizes))  # fp32 views at odd offsets
    norm2 = ops.clip_grad_norm(grads, max_norm, norm_type=kind, out=outs)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(grads, before))
    check_clip(before, outs, norm, max_norm, kind)
    norm3 = ops.clip_grad_norm(grads, max_norm, norm_type=kind)  # in place
    assert torch.equal(norm, norm3)
    check_clip(before, grads, norm, max_norm, kind)
    if max_norm > norm.item():
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert all(torch.equal(o.to(g.dtype), g) for o, g in zip(outs, grads))


def test_clip_layouts():
    g = gen(31)
    a = torch.randn(300, 40, generator=g, device=DEV).t()          # dense, another order
    b = torch.randn(64, 50, generator=g, device=DEV)[:, 3:20]      # gaps between the rows
    c = torch.randn(1001, generator=g, device=DEV)[1:]             # off a 16-byte boundary
    gap = b._base.clone()
    before = [t.clone() for t in (a, b, c)]
    o = [torch.empty(40, 300, device=DEV), torch.empty(64, 17, device=DEV), torch.empty(2000, device=DEV)[::2]]
    norm = ops.clip_grad_norm([a, b, c], 1.0, out=o)
    check_clip(before, o, norm, 1.0, 2.0)
    ops.clip_grad_norm([a, b, c], 1.0)
    check_clip(before, [a, b, c], norm, 1.0, 2.0)
    gap[:, 3:20] = b
    assert torch.equal(gap, b._base)  # the memory between the rows is untouched


@pytest.mark.parametrize("v, dtype", [(1e30, F32), (1e-30, F32), (3e38, F32), (6e4, F16), (1e-40, F32)])
def test_clip_does_not_overflow_before_the_norm(v, dtype):
    t = torch.full((10_000,), v, dtype=dtype, device=DEV)
    before = t.clone()
    norm = ops.clip_grad_norm([t], 1.0)
    want = before[0].double() * 100
    if want > torch.finfo(F32).max:  # the norm itself does not fit 32 bits: reported inf, the gradients clipped by it
        assert norm.isinf()
    else:
        check(norm, want, 1.001 * U * want + TINY[F32], "norm")
    check_w = before.double() * min(1.0, 1.0 / (want.item() + 1e-6))
    check(t, check_w, 2.001 * U * check_w + stored(check_w, dtype), "clipped")


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_clip_non_finite_norms_spread_as_in_torch(kind, bad):
    t = torch.ones(30_000, device=DEV)
    t[12_345] = bad
    p = torch.nn.Parameter(torch.zeros_like(t))
    p.grad = t.clone()
    want = torch.nn.utils.clip_grad_norm_([p], 1.0, kind)
    norm = ops.clip_grad_norm([t], 1.0, kind)
    assert torch.equal(norm.isnan(), want.isnan()) and torch.equal(norm.isinf(), want.isinf())
    check(t, p.grad, 0.0, "clipped")
    with pytest.raises(RuntimeError, match="non-finite"):
        q = torch.nn.Parameter(torch.zeros_like(t))
        q.grad = torch.full_like(t, bad)
        optim.clip_grad_norm_([q], 1.0, kind, error_if_nonfinite=True)
    assert torch.equal(q.grad.isfinite(), torch.zeros_like(t, dtype=torch.bool))  # raised before anything changed


def test_clip_of_empty_tensors():
    norm = ops.clip_grad_norm([torch.empty(0, device=DEV), torch.empty(3, 0, device=DEV)], 1.0)
    assert norm.item() == 0.0 and norm.device.type == "cuda"


def test_clip_grad_norm_of_parameters():
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((30, 40), (7,), (1,))]
    for p in ps[:2]:
        p.grad = torch.randn(p.shape, generator=gen(32), device=DEV)
    before = [p.grad.clone() for p in ps[:2]]
    norm = optim.clip_grad_norm_((p for p in [*ps, ps[0]]), 1.0)  # one without a gradient, one twice
    check_clip(before, [p.grad for p in ps[:2]], norm, 1.0, 2.0)


def test_clip_counts_as_an_in_place_change():
    """A backward that saved a gradient must not run with its clipped values, as with torch's own in-place calls."""
    flat = torch.randn(600, generator=gen(36), device=DEV)
    a, b = torch.randn(600, generator=gen(37), device=DEV), flat[100:].view(20, 25)
    x = torch.ones(600, device=DEV, requires_grad=True)
    for fn in (lambda: ops.clip_grad_norm([a], 0.5), lambda: ops.clip_grad_norm([b.clone()], 0.5, out=[a[:500].view(20, 25)]),
               lambda: ops.clip_grad_norm([a, b.t()[:, ::2]], 0.5)):
        y = (x * a).sum()
        fn()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    y = (x * flat).sum()
    ops.clip_grad_norm([b], 0.5)  # a view's change is its base's
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (x * a).sum()
    ops.clip_grad_norm([a], None)  # the norm alone changes nothing
    ops.clip_grad_norm([a], 0.5, out=[torch.empty_like(a)])
    y.backward()
    with torch.inference_mode():
        t = torch.ones(40, device=DEV)
        ops.clip_grad_norm([t], 1.0)
    p = torch.nn.Parameter(torch.zeros(40, device=DEV))
    p.grad = torch.ones(40, device=DEV)
    before = p.grad._version
    optim.clip_grad_norm_([p], 1.0)
    assert p.grad._version > before


def test_clip_offsets_beyond_32_bits():
    n = 2 ** 31 + 5
    t = torch.zeros(n, dtype=BF16, device=DEV)
    t[-3:] = 2.0
    t[0] = 2.0
    norm = ops.clip_grad_norm([t], 2.0)
    assert norm.item() == 4.0
    assert (t[-3:] == 1.0).all() and t[0] == 1.0 and not t[1:-3].any()


def test_clip_captured_and_replayed():
    sizes, types = [70_000, 33, 5000] * 60, [F32, BF16, F32] * 60  # two launches' lists
    grads = clip_case(sizes, types, 33)
    outs = [torch.empty(s, device=DEV) for s in sizes]
    ops.clip_grad_norm(grads, 1.0, out=outs)
    graphs, norms = [], []
    for _ in range(2):  # two graphs over the same tensors: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(ops.clip_grad_norm(grads, 1.0, out=outs))
        graphs.append(graph)
    for k in range(3):
        for g, new in zip(grads, clip_case(sizes, types, 34 + k, scale=10.0 ** (k - 1))):
            g.copy_(new)
        want = [torch.empty_like(o) for o in outs]
        wn = ops.clip_grad_norm(grads, 1.0, out=want)
        for graph, norm in zip(graphs, norms):
            for o in outs:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, wn) and all(torch.equal(a, b) for a, b in zip(outs, want)), k


# ---------------------------------------------------------------------------------------------
# 4-bit rows
def exact_quantize(x, group):
    """Codes and scales by the definition in 64 bits: bf16(max / 7) and x / scale, each rounded to nearest even."""
    n, H = x.shape
    ng = -(-H // group)
    pad = torch.nn.functional.pad(x.double(), (0, ng * group - H)).view(n, ng, group)
    s = pad.abs().amax(2) / 7
    e = torch.floor(torch.log2(s.clamp(min=2.0 ** -126)))
    step = torch.exp2(e - 7)
    s = torch.round(s / step) * step  # (torch.round: ties to even)
    c = torch.where(s.unsqueeze(2) > 0, torch.round(pad / s.unsqueeze(2)), 0.0).clamp(-7, 7)
    return (c * s.unsqueeze(2)).view(n, -1)[:, :H], s


INT4 = [(1, 1, 32), (5, 31, 32), (16, 32, 64), (17, 33, 32), (40, 100, 64), (1000, 128, 128), (333, 256, 32),
        (50, 300, 128), (19, 4096, 64)]


@pytest.mark.parametrize("n, H, group", INT4)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_int4_quantize_is_the_definition(n, H, group, dtype):
    x = torch.randn(n, H, generator=gen(40), device=DEV)
    x[0] = (torch.arange(H, device=DEV) % 15 - 7) * 0.5  # quotients that are integers and halves
    if n > 2:
        x[1] = 0.0
        x[2] *= 1e-3
    x = x.to(dtype)
    rows = ops.Int4Rows.quantize(x, group)
    want, _ = exact_quantize(x, group)
    assert torch.equal(rows.dequantize().double(), want)
    # a row's group is off by at most half a step of its scale (and its clamp: the scale's own rounding, 7 2^-8)
    assert ((want - x.double()).abs() <= 0.5001 * x.double().abs().amax(1, keepdim=True) / 7 * (1 + 2 ** -7)
            + 7 * 2.0 ** -8 * x.double().abs().amax(1, keepdim=True) / 7).all()


def test_int4_quantize_ties_and_extremes():
    x = torch.zeros(8, 32, device=DEV)
    x[0] = torch.linspace(-7, 7, 32, device=DEV)
    x[1, :4] = torch.tensor([7.0, 0.5, 1.5, -2.5], device=DEV)  # scale 1: ties to even
    x[2] = 1e38
    x[3] = 1e-37
    x[4, 3] = math.nan
    x[5, 3] = math.inf
    x[6, 0] = 7 * (1 + 2.0 ** -8)  # the quotient is a bf16 tie, exactly
    x[7, 0] = 1e-42  # a scale below every bf16 number
    got = ops.Int4Rows.quantize(x, 32).dequantize()
    assert got[1, :4].tolist() == [7.0, 0.0, 2.0, -2.0]
    want, _ = exact_quantize(x[[0, 2, 3, 6]], 32)
    assert torch.equal(got[[0, 2, 3, 6]].double(), want)
    assert got[4].isnan().all() and got[5].isnan().all()
    assert got[7].abs().max() <= 1e-42


def check_scores(got, q, values, scale_mass, nblk):
    """values (n, H) 64 bit.  Per 32 columns three chains of 32 exact products added in fp32 (the adders may
    truncate: a whole step each), the three joined; then one product and one sum per block; q itself
    to 2^-27 of its largest element."""
    q = q.double()
    want = q @ values.t()
    mass = q.abs() @ values.abs().t()
    bound = (2 * (3 * 32 + 3) + nblk + 4) * U * mass
    bound = bound + 2.0 ** -27 * q.abs().amax(1, keepdim=True) * values.abs().sum(1)
    check(got, want, bound + TINY[F32], "scores")


@pytest.mark.parametrize("n, H, group", INT4)
@pytest.mark.parametrize("nq, dtype", [(1, F32), (4, BF16), (5, F16), (16, F32), (33, F32), (64, BF16), (70, F32)])
def test_int4_scores_against_plain(n, H, group, nq, dtype):
    g = gen(41)
    codes = torch.randint(-8, 8, (n, H), generator=g, device=DEV, dtype=torch.int8)
    scales = (torch.rand(n, -(-H // group), generator=g, device=DEV) + 0.1).to(BF16)
    rows = ops.Int4Rows.from_codes(codes, scales, group)
    values = codes.double() * scales.double().repeat_interleave(group, 1)[:, :H]
    assert torch.equal(rows.dequantize().double(), values)
    q = torch.randn(nq, H, generator=g, device=DEV).to(dtype)
    got = ops.int4_scores(q, rows)
    assert got.shape == (nq, n) and got.dtype == F32
    check_scores(got, q, values, scales, -(-H // 32))
    assert torch.equal(ops.int4_scores(q, rows), got)


@pytest.mark.parametrize("n, H, group, nq", [(70_001, 1024, 128, 9), (70_001, 1024, 32, 20), (33_000, 256, 64, 32),
                                            (66_000, 256, 32, 64), (40_000, 36, 32, 3)])
def test_int4_scores_of_a_long_index(n, H, group, nq):
    """Enough rows for the larger workgroups, whose waves share the query operands."""
    g = gen(47)
    codes = torch.randint(-8, 8, (n, H), generator=g, device=DEV, dtype=torch.int8)
    scales = (torch.rand(n, -(-H // group), generator=g, device=DEV) + 0.1).to(BF16)
    rows = ops.Int4Rows.from_codes(codes, scales, group)
    values = codes.double() * scales.double().repeat_interleave(group, 1)[:, :H]
    assert torch.equal(rows.dequantize().double(), values)
    q = torch.randn(nq, H, generator=g, device=DEV)
    check_scores(ops.int4_scores(q, rows), q, values, scales, -(-H // 32))


def test_int4_scores_strides_and_shapes():
    g = gen(42)
    x = torch.randn(100, 64, generator=g, device=DEV)
    rows = ops.Int4Rows.quantize(torch.nn.functional.pad(x, (3, 5))[:, 3:67], 32)  # rows 72 apart, off alignment
    assert torch.equal(rows.dequantize(), ops.Int4Rows.quantize(x, 32).dequantize())
    wide = torch.randn(6, 75, generator=g, device=DEV)
    q = wide[:, 5:69]
    want = ops.int4_scores(q.contiguous(), rows)
    assert torch.equal(ops.int4_scores(q, rows), want)
    assert torch.equal(ops.int4_scores(q.t().contiguous().t(), rows), want)
    assert torch.equal(ops.int4_scores(q[2], rows), ops.int4_scores(q[2:3], rows))
    assert torch.equal(ops.int4_scores(q[:1].expand(5, 64), rows)[4], ops.int4_scores(q[:1].repeat(5, 1), rows)[4])
    assert ops.int4_scores(q[:0], rows).shape == (0, 100)
    empty = ops.Int4Rows.quantize(x[:0], 32)
    assert ops.int4_scores(q, empty).shape == (6, 0) and empty.dequantize().shape == (0, 64)


def test_int4_scores_query_scales_and_non_finite():
    g = gen(43)
    codes = torch.randint(-8, 8, (50, 96), generator=g, device=DEV, dtype=torch.int8)
    scales = (torch.rand(50, 3, generator=g, device=DEV) + 0.1).to(BF16)
    scales[7, 1] = math.nan
    scales[9, 1] = math.inf
    rows = ops.Int4Rows.from_codes(codes, scales, 32)
    fine = torch.ones(50, dtype=torch.bool, device=DEV)
    fine[[7, 9]] = False
    values = codes.double() * scales.double().repeat_interleave(32, 1)
    for nq in (4, 12, 40):
        q = torch.randn(nq, 96, generator=g, device=DEV)
        q[0] *= 1e-30
        q[1] *= 1e30
        q[2, 5] = math.nan
        q[3] = 0.0
        got = ops.int4_scores(q, rows)
        ok = torch.ones(nq, dtype=torch.bool, device=DEV)
        ok[2] = False
        check_scores(got[ok][:, fine], q[ok], values[fine], scales, 3)
        assert got[2].isnan().all() and got[:, 7].isnan().all()
        assert not got[4:, 9].isfinite().any()
        assert not got[3, fine].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nq", [1, 4, 12, 40])
@pytest.mark.parametrize("ratio", [300.0, 3e4, 1e6])
def test_int4_scores_beside_a_dominant_element(ratio, nq, dtype):
    """One query element far above the others, at a column whose codes are zero: nothing of the others is lost but
    what lies below 2^-39 of it."""
    g = gen(48)
    n, H = 300, 96
    codes = torch.randint(-8, 8, (n, H), generator=g, device=DEV, dtype=torch.int8)
    codes[:, 37] = 0
    codes[0] = 0
    codes[0, 70] = 7  # one product alone: exact but for the terms' sum and two roundings
    scales = (torch.rand(n, 3, generator=g, device=DEV) + 0.1).to(BF16)
    values = codes.double() * scales.double().repeat_interleave(32, 1)
    q = (torch.randn(nq, H, generator=g, device=DEV) / ratio).to(dtype)
    q[:, 37] = 1.0
    got = ops.int4_scores(q, ops.Int4Rows.from_codes(codes, scales, 32))
    q = q.double()
    want, mass = q @ values.t(), q.abs() @ values.abs().t()
    lost = 2.0 ** -39 * values.abs().sum(1)
    # (2 (3 x 32 + 3) + 3 + 4) u as in check_scores, what the terms leave out beside it
    check(got, want, 205 * U * mass + lost, "scores")
    check(got[:, 0], want[:, 0], 10 * U * want[:, 0].abs() + lost[0], "one product")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nq, H", [(4, 80), (12, 80), (40, 80), (6, 2100), (70, 300)])
def test_int4_scores_of_infinite_queries(nq, H, dtype):
    """Infinities as in a product of floats: signed by their codes, NaN at a zero code or against another one; the other
    queries of the batch and finite elements beside them, however large, change nothing."""
    g = gen(49)
    n = 200
    codes = torch.randint(-8, 8, (n, H), generator=g, device=DEV, dtype=torch.int8)
    codes[:20, 7] = 0
    scales = (torch.rand(n, -(-H // 64), generator=g, device=DEV) + 0.1).to(BF16)
    scales[30, 0] = 0.0
    values = codes.double() * scales.double().repeat_interleave(64, 1)[:, :H]
    rows = ops.Int4Rows.from_codes(codes, scales, 64)
    q = torch.randn(nq, H, generator=g, device=DEV).to(dtype)
    plain = ops.int4_scores(q, rows)
    q[0, 7] = math.inf
    q[0, 70] = torch.finfo(dtype).max
    q[1, [7, 60]] = torch.tensor([math.inf, -math.inf], device=DEV, dtype=dtype)
    q[2, 7] = math.nan
    q[3] = -math.inf
    got = ops.int4_scores(q, rows)
    want = (q.double().cpu() @ values.cpu().t()).to(DEV)
    assert torch.equal(got[:4].isnan(), want[:4].isnan())
    check(got[:4], want[:4], 0.0, "infinite")  # nothing is finite there
    assert got[0].isinf().sum() > 150 and got[1].isinf().any() and torch.equal(got[4:], plain[4:])


def test_int4_scores_of_queries_that_need_a_gradient():
    rows = ops.Int4Rows.quantize(torch.randn(100, 48, generator=gen(50), device=DEV))
    q = torch.randn(3, 48, generator=gen(51), device=DEV, requires_grad=True)
    scores = ops.int4_scores(q, rows)
    assert torch.equal(scores, ops.int4_scores(q.detach(), rows))
    assert torch.equal(ops.topk_rows(scores, 4)[0], scores.topk(4, dim=1).values)
    with pytest.raises(RuntimeError, match="no gradient"):
        (scores.sum() + q.sum()).backward()


def test_int4_scores_offsets_beyond_32_bits():
    n, H = 34_000_000, 256  # 4.35 GB of codes
    codes = torch.zeros(n, H, dtype=torch.int8, device=DEV)
    codes[-5:] = torch.arange(-5, 0, device=DEV, dtype=torch.int8).unsqueeze(1)
    rows = ops.Int4Rows.from_codes(codes, torch.ones(n, H // 128, dtype=BF16, device=DEV), 128)
    del codes
    got = ops.int4_scores(torch.ones(1, H, device=DEV), rows)
    assert got[0, -5:].tolist() == [-5.0 * H, -4.0 * H, -3.0 * H, -2.0 * H, -1.0 * H]
    assert not got[0, :-5].any()


def test_int4_scores_captured_and_on_another_stream():
    rows = ops.Int4Rows.quantize(torch.randn(1000, 128, generator=gen(44), device=DEV), 64)
    q = torch.randn(3, 128, generator=gen(45), device=DEV)
    ops.int4_scores(q, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.int4_scores(q, rows)
    for k in range(3):
        q.copy_(torch.randn(3, 128, generator=gen(46 + k), device=DEV))
        want = ops.int4_scores(q, rows)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.int4_scores(q, rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


# ---------------------------------------------------------------------------------------------
# the operators together: a fine-tuning step and the index that serves its tower
class TokenTower(torch.nn.Module):
    """A foreign tower that pools its token rows itself (softmax-weighted by a learned direction)."""

    def __init__(self, embedding, hidden_dim):
        super().__init__()
        self.embedding = embedding
        self.gate = torch.nn.Parameter(torch.randn(embedding.embedding_dim) * 0.1)
        self.out = torch.nn.Linear(embedding.embedding_dim, hidden_dim)

    def forward(self, ids):
        rows = self.embedding(ids)
        a = (rows * self.gate).sum(-1).masked_fill(ids == 0, -1e9).softmax(-1)
        return torch.nn.functional.normalize(self.out((a.unsqueeze(-1) * rows).sum(1)), dim=-1)


def token_model(seed):
    torch.manual_seed(seed)
    emb = tt.embeddings.build("lookup", vocab_size=300, embedding_dim=64, scale=8.0)
    with torch.no_grad():
        emb.embedding.weight.mul_(0.125)
    return tt.TwoTower(TokenTower(emb, 128), tied_weights=True)


def triplets(B, L, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(1, 300, (3, B, L), generator=g)
    ids[:, :, L // 2:] *= (torch.rand(3, B, L - L // 2, generator=g) > 0.4)
    return ids


@pytest.mark.parametrize("B", [16, 400])  # 960 and 24,000 tokens a step: both forms of the lookup's gradient
def test_fine_tuning_step_against_64_bits(B):
    model, ref64 = token_model(50), token_model(50).double()
    frozen = token_model(51).to(DEV)
    model.to(DEV)
    ids = triplets(B, 20, 52)
    gpu = ids.to(DEV)
    with torch.no_grad():
        ref = losses.preference_margin(*(frozen.encode_query(t) for t in gpu))
    loss_fn = losses.build("preference", beta=0.5, ref_margin=ref)
    opt = optim.AdamW(model.parameters(), lr=1e-3, capturable=True)
    step = tt.TrainStep(model, loss_fn, opt, max_grad_norm=0.05)
    with _lib.record_calls() as calls:
        loss = step(*gpu)
    assert {"tt_lookup_fwd", "tt_lookup_bwd", "tt_preference_fwd", "tt_preference_bwd", "tt_clip_grads"} <= calls
    # the same step in 64 bits on the CPU
    q, p, n = (ref64.query_tower(t) for t in ids)
    h = (q * (p - n)).sum(-1) / 0.1 - ref.cpu().double()[:, 0]
    want = torch.nn.functional.softplus(-0.5 * h).mean()
    want.backward()
    params = [x for x in ref64.parameters()]
    norm = torch.nn.utils.clip_grad_norm_(params, 0.05)
    # fp32 towers: some 1e-6 relative in the margins (|h| up to 20), less in their means
    assert abs(loss.item() - want.item()) < 1e-5 * max(1.0, want.item())
    assert abs(step.grad_norm.item() - norm.item()) < 1e-4 * norm.item()
    for a, b in zip(model.parameters(), params):
        assert (a.grad.cpu().double() - b.grad).norm() <= 1e-4 * b.grad.norm()
    total = torch.cat([x.grad.flatten() for x in model.parameters()]).double().norm().item()
    assert abs(total - min(0.05, norm.item())) < 1e-5


def test_captured_fine_tuning_equals_eager():
    batches = [triplets(32, 20, 60 + k).to(DEV) for k in range(6)]
    runs = []
    for graph in (False, True):
        model = token_model(53).to(DEV)
        opt = optim.AdamW(model.parameters(), lr=1e-2, capturable=True)
        step = tt.TrainStep(model, losses.build("preference", beta=0.5), opt, graph=graph, max_grad_norm=0.1)
        runs.append(([step(*b).item() for b in batches], [x.detach().clone() for x in model.parameters()]))
    # one arithmetic, but library GEMMs may pick another form under capture
    assert all(abs(a - b) < 1e-4 for a, b in zip(runs[0][0], runs[1][0]))
    for a, b in zip(runs[0][1], runs[1][1]):
        assert (a - b).norm() <= 1e-3 * b.norm()


@pytest.mark.parametrize("graph", [False, True])
def test_each_batch_trains_against_its_own_reference(graph):
    """Margins and masks of the batch, passed to the step: eager and captured steps against the loss of that batch, in
    any order of shapes, with and without them, from tensors of other layouts and types."""
    model = token_model(63).to(DEV)
    opt = optim.AdamW(model.parameters(), lr=0.0, weight_decay=0.0, capturable=True)  # the parameters stay
    loss_fn = losses.build("preference", beta=0.5)
    step = tt.TrainStep(model, loss_fn, opt, graph=graph, eager_steps=1, max_grad_norm=1e9)
    g = gen(64)
    batches = []
    for k, B in enumerate((12, 12, 20, 12, 20, 12)):
        ids = triplets(B, 20, 65 + k).to(DEV)
        kw = {"ref_margin": torch.randn(B, 2, generator=g, device=DEV)[:, 1],
              "mask": (torch.rand(1, B, generator=g, device=DEV) > 0.3).t()}
        batches.append((ids, kw if k != 3 else {"mask": kw["mask"], "ref_margin": None}))
    batches += [(ids, {"ref_margin": kw["ref_margin"]}) for ids, kw in batches[:2]] + [(batches[0][0], {})]
    batches += [(ids, dict(reversed(kw.items()))) for ids, kw in batches[:2]]  # the names' order means nothing

    def plain(ids, kw):  # (numbers alone: no graph of the parameters may live while a step is captured)
        want = loss_fn(*model(*ids), **kw)
        grads = torch.autograd.grad(want, list(model.parameters()))
        return want.item(), torch.cat([x.flatten() for x in grads]).norm().item()

    for ids, kw in batches * 2:
        loss = step(*ids, **kw).item()
        want, norm = plain(ids, kw)
        assert abs(loss - want) <= 1e-5 * max(1.0, want)
        assert abs(step.grad_norm.item() - norm) <= 1e-4 * norm


def test_no_capture_beside_a_live_graph_of_the_parameters():
    model = token_model(66).to(DEV)
    opt = optim.AdamW(model.parameters(), lr=0.0, weight_decay=0.0, capturable=True)
    loss_fn = losses.build("preference", beta=0.5)
    step = tt.TrainStep(model, loss_fn, opt, graph=True, eager_steps=1)
    ids = triplets(12, 20, 67).to(DEV)
    first = step(*ids).item()
    held = loss_fn(*model(*ids))
    with pytest.raises(RuntimeError, match="still alive"):
        step(*ids)
    held = held.item()
    assert abs(step(*ids).item() - first) <= 1e-5 and abs(step(*ids).item() - held) <= 1e-5
    held = loss_fn(*model(*ids))  # a recorded step needs no more
    assert abs(step(*ids).item() - first) <= 1e-5


def test_captured_clipping_keeps_each_graphs_norm():
    model = token_model(58).to(DEV)
    opt = optim.AdamW(model.parameters(), lr=0.0, weight_decay=0.0, capturable=True)  # the parameters stay
    step = tt.TrainStep(model, losses.build("preference", beta=0.5), opt, graph=True, eager_steps=1, max_grad_norm=0.1)
    eager = tt.TrainStep(model, losses.build("preference", beta=0.5), opt, max_grad_norm=0.1)
    small, large = triplets(8, 20, 61).to(DEV), triplets(24, 20, 62).to(DEV)
    step(*small)
    for b in (small, large, small, large, small):
        step(*b)
        got = step.grad_norm.item()
        eager(*b)
        assert abs(got - eager.grad_norm.item()) <= 1e-4 * got


def test_clipping_beside_the_hand_written_tower_head():
    """The mean-pool tower's head may form its weight gradients on a side stream: the norm needs them all."""
    def build():
        torch.manual_seed(54)
        emb = tt.embeddings.build("lookup", vocab_size=500, embedding_dim=256)
        return tt.build_two_tower("mean", emb, hidden_dim=256, tied_weights=True).to(DEV)

    ids = triplets(64, 12, 55).to(DEV)
    ref = build()
    loss = losses.build("preference", beta=0.5)(*ref(*ids))
    loss.backward()
    want = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.01)
    model = build()
    opt = optim.AdamW(model.parameters(), capturable=True)
    step = tt.TrainStep(model, losses.build("preference", beta=0.5), opt, max_grad_norm=0.01)
    step(*ids)
    assert abs(step.grad_norm.item() - want.item()) <= 1e-5 * want.item()
    for a, b in zip(model.parameters(), ref.parameters()):
        assert (a.grad - b.grad).norm() <= 1e-5 * b.grad.norm()


@pytest.mark.parametrize("group", [32, 64])
def test_search_with_a_4_bit_index(group, tmp_path):
    model = token_model(56).to(DEV)
    docs = triplets(500, 20, 57)[0].to(DEV)
    plain = tt.search.TwoTowerSearch(model)
    plain.index_document_ids(docs)
    s = tt.search.TwoTowerSearch(model, index_dtype="int4", index_group=group)
    s.index_document_ids(docs)
    assert s.document_embeddings is None and s.index.n == 500
    queries = docs[:9]
    scores, idx = s.search_ids(queries, top_k=5)
    # the top of the scores against the index's own values, in 64 bits
    q = torch.nn.functional.normalize(plain.encode_queries(queries).double(), dim=-1)
    want = q @ s.index.dequantize().double().t()
    top = want.topk(5, dim=1).values
    assert (scores.double() - top).abs().max() <= 400 * U * 10
    assert torch.equal(idx[:, 0], torch.arange(9, device=DEV))  # a document is its own nearest
    # 4 bits: a unit row's values are off by at most half a step of max / 7 each
    full, _ = plain.search_ids(queries, top_k=5)
    assert (scores - full).abs().max() < 0.2
    s.save_index(str(tmp_path / "index.pt"))
    r = tt.search.TwoTowerSearch(model)
    r.load_index(str(tmp_path / "index.pt"))
    again, idx2 = r.search_ids(queries, top_k=5)
    r.index_document_ids(docs[:50])  # its own kind of index replaces the loaded one
    assert r.index is None and r.search_ids(queries, top_k=60)[0].shape == (9, 50)
    assert torch.equal(again, scores) and torch.equal(idx2, idx)


def test_empty_calls():
    """No token, pair, element, query or row: empty results, a loss and a norm of 0."""
    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    out = ops.embedding_lookup(w, torch.empty(0, 3, dtype=torch.int64, device=DEV))
    assert out.shape == (0, 3, 8) and not torch.autograd.grad(out.sum(), w)[0].any()
    q, p, n = (torch.empty(s, device=DEV, requires_grad=True) for s in ((0, 8), (0, 8), (0, 2, 8)))
    loss = losses.preference_loss(q, p, n)
    assert loss.item() == 0.0 and [g.shape for g in torch.autograd.grad(loss, (q, p, n))] == [q.shape, p.shape, n.shape]
    assert losses.preference_margin(q, p, n).shape == (0, 2)
    empty = torch.empty(0, device=DEV)
    assert ops.clip_grad_norm([empty, empty.clone()], 1.0).item() == 0.0 == ops.clip_grad_norm([empty], None).item()
    rows = ops.Int4Rows.quantize(torch.empty(0, 40, device=DEV))
    assert ops.int4_scores(torch.randn(3, 40, device=DEV), rows).shape == (3, 0) and rows.dequantize().shape == (0, 40)
    rows = ops.Int4Rows.quantize(torch.randn(4, 40, device=DEV))
    assert ops.int4_scores(torch.empty(0, 40, device=DEV), rows).shape == (0, 4)
