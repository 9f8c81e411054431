"""CPU: argument checks of the token lookup, preference loss, gradient clipping and 4-bit index operators, at the
Python entry points and at the C ABI (every refused call returns before a launch), and the loss
formulas' derivatives against differences."""
import ctypes
import math

import pytest
import torch

import twotower_amd as tt
from twotower_amd import _lib, losses, ops, optim

P = 4096  # a pointer-shaped value; refused calls never read it


# ---------------------------------------------------------------------------------------------
# Python entry points
@pytest.mark.parametrize("kw, err, msg", [
    (dict(weight=torch.zeros(4)), ValueError, "weight must be"),
    (dict(weight=torch.zeros(0, 4)), ValueError, "weight must be"),
    (dict(weight=torch.zeros(4, 4, dtype=torch.float64)), TypeError, "weight must be float32"),
    (dict(ids=torch.zeros(2, dtype=torch.int16)), TypeError, "token ids must be"),
    (dict(weight=torch.zeros(4, 8).t()), ValueError, "rows must be contiguous"),
    (dict(weight=torch.zeros(1, 4).expand(5, 4)), ValueError, "must not overlap"),
    (dict(out_dtype=torch.float64), TypeError, "out_dtype"),
    (dict(weight=torch.zeros(4, 4, dtype=torch.bfloat16), out_dtype=torch.float32), TypeError, "out_dtype"),
    (dict(padding_idx=4), ValueError, "padding_idx"),
    (dict(padding_idx=-5), ValueError, "padding_idx"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_lookup_refusals(kw, err, msg):
    args = dict(weight=torch.zeros(4, 4), ids=torch.zeros(2, 3, dtype=torch.int64))
    args.update(kw)
    with pytest.raises(err, match=msg):
        ops.embedding_lookup(**args)


def test_lookup_of_a_column_sharded_table_is_refused(monkeypatch):
    w = torch.nn.Parameter(torch.zeros(4, 4))
    w._tt_column = type("Col", (), {"stale": True})()
    monkeypatch.setattr(_lib, "same_device", lambda *a: None)
    with pytest.raises(RuntimeError, match="column-sharded"):
        ops.embedding_lookup(w, torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("kw, err, msg", [
    (dict(p=torch.zeros(3, 5)), ValueError, "q and p must both be"),
    (dict(q=torch.zeros(3, 4, 1)), ValueError, "q and p must both be"),
    (dict(n=torch.zeros(2, 4)), ValueError, "n must be"),
    (dict(n=torch.zeros(3, 0, 4)), ValueError, "n must be"),
    (dict(n=torch.zeros(3, 2, 5)), ValueError, "n must be"),
    (dict(p=torch.zeros(3, 4, dtype=torch.bfloat16)), TypeError, "one type"),
    (dict(ref_margin=torch.zeros(3)), ValueError, "ref_margin must be"),
    (dict(ref_margin=torch.zeros(3, 2, dtype=torch.int64)), TypeError, "ref_margin must be"),
    (dict(mask=torch.ones(3, 1, dtype=torch.bool)), ValueError, "mask must be"),
    (dict(mask=torch.ones(3, 2)), TypeError, "mask must be bool"),
    (dict(beta=0.0), ValueError, "beta and temperature"),
    (dict(temperature=-1.0), ValueError, "beta and temperature"),
    (dict(temperature=math.nan), ValueError, "beta and temperature"),
    (dict(label_smoothing=1.0), ValueError, "label_smoothing"),
    (dict(label_smoothing=0.1, loss_type="squared"), ValueError, "label_smoothing"),
    (dict(loss_type="hinge"), ValueError, "loss_type"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_preference_refusals(kw, err, msg):
    args = dict(q=torch.zeros(3, 4), p=torch.zeros(3, 4), n=torch.zeros(3, 2, 4))
    args.update(kw)
    with pytest.raises(err, match=msg):
        losses.preference_loss(args.pop("q"), args.pop("p"), args.pop("n"), **args)


def test_preference_is_built_by_name():
    f = losses.build("preference", beta=0.5)
    assert f.func is losses.preference_loss and f.keywords == {"beta": 0.5}
    assert tt.preference_loss is losses.preference_loss


@pytest.mark.parametrize("grads, kw, err, msg", [
    ([torch.ones(3)], dict(max_norm=-1.0), ValueError, "max_norm"),
    ([torch.ones(3)], dict(max_norm=math.nan), ValueError, "max_norm"),
    ([torch.ones(3)], dict(norm_type=1.0), ValueError, "norm_type"),
    ([torch.ones(3)], dict(out=[]), ValueError, "out tensors"),
    ([torch.ones(3)], dict(out=[torch.ones(4)]), ValueError, "out 0 has shape"),
    ([torch.ones(3)], dict(out=[torch.ones(3, dtype=torch.bfloat16)]), TypeError, "gradient 0"),
    ([torch.ones(3)], dict(max_norm=None, out=[torch.ones(3)]), ValueError, "out needs a max_norm"),
    ([torch.ones(3, dtype=torch.float64)], {}, TypeError, "gradient 0"),
    ([torch.ones(3, 3).to_sparse()], {}, RuntimeError, "sparse"),
    ([torch.ones(1, 3).expand(4, 3)], {}, ValueError, "share memory"),
    ([torch.ones(3)], {}, RuntimeError, "no CPU fallback"),
])
def test_clip_refusals(grads, kw, err, msg):
    args = dict(max_norm=1.0)
    args.update(kw)
    with pytest.raises(err, match=msg):
        ops.clip_grad_norm(grads, **args)


def test_clip_refuses_the_same_memory_twice():
    t = torch.ones(8)
    with pytest.raises(ValueError, match="written twice"):
        ops.clip_grad_norm([t, t.view(2, 4)], 1.0)


def test_clip_refuses_an_out_that_is_another_gradient():
    a, b = torch.ones(8), torch.ones(8)
    with pytest.raises(ValueError, match="memory of another gradient"):
        ops.clip_grad_norm([a, b], 1.0, out=[b, a])
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # its own gradient's memory is fine
        ops.clip_grad_norm([a, b], 1.0, out=[a, torch.ones(8)])


def test_clip_refuses_tensors_that_overlap_in_part():
    t, h = torch.ones(40), torch.ones(40, dtype=torch.bfloat16)
    other = torch.ones(40)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            ops.clip_grad_norm(*args, 1.0, **kw)

    def taken(*args, **kw):  # (as far as the check for GPU tensors, after the others)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            ops.clip_grad_norm(*args, 1.0, **kw)

    refused("written twice", [t[:20], t[19:]])
    refused("written twice", [t[30:], other, t[5:31]])
    refused("written twice", [t, t[7:9]])
    refused("written twice", [other, other.clone()], out=[t[:40], t.view(2, 20).view(40)])
    refused("memory of another gradient", [t[:20], other[:20]], out=[other[20:], t[10:30]])
    refused("memory of another gradient", [t[:20]], out=[t[1:21]])
    refused("memory of another gradient", [h[:20]], out=[h.view(torch.float32)])
    taken([t[20:], t[:20], other])
    taken([t[:20], h], out=[t[20:], other])
    taken([t[:20], t[20:]], out=[other[20:], other[:20]])
    taken([t[:20], t[20:]], out=[t[:20], t[20:]])
    taken([t[20:], t[:0], other[:0], t[:20]], out=[t[20:], t[:0], t[:0], t[:20]])  # nothing to write


def test_clip_of_nothing_and_of_a_fused_table():
    assert ops.clip_grad_norm([], 1.0).item() == 0.0
    assert optim.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0).item() == 0.0
    w = torch.nn.Parameter(torch.ones(2, 2))
    w._tt_deferred = ops.DeferredTableGrad()
    w._tt_deferred.parts.append(("part",))
    with pytest.raises(RuntimeError, match="factored form"):
        optim.clip_grad_norm_([w], 1.0)


def test_clip_refuses_parameters_that_are_stepped_inside_backward():
    """Nothing of their gradients is left to clip, and the norm would leave them out."""
    emb = tt.embeddings.build("lookup", vocab_size=20, embedding_dim=8)
    model = tt.build_two_tower("mean", emb, hidden_dim=16, tied_weights=True)
    opt = torch.optim.AdamW(model.parameters())
    assert optim.clip_grad_norm_(model.parameters(), 1.0).item() == 0.0
    (table,) = optim.fuse_table_update(opt, model)
    with pytest.raises(RuntimeError, match="stepped inside backward"):
        optim.clip_grad_norm_(model.parameters(), 1.0)
    table.release()
    dense = optim.fuse_dense_update(opt, model)
    with pytest.raises(RuntimeError, match="stepped inside backward"):
        optim.clip_grad_norm_(model.parameters(), 1.0)
    dense.release()
    assert optim.clip_grad_norm_(model.parameters(), 1.0).item() == 0.0


def test_train_step_refuses_clipping_a_fused_table():
    emb = tt.embeddings.build("lookup", vocab_size=20, embedding_dim=8)
    model = tt.build_two_tower("mean", emb, hidden_dim=16, tied_weights=True)
    opt = optim.AdamW(model.parameters(), fused_tables=True, tables=[emb])
    loss = losses.build("preference")
    with pytest.raises(ValueError, match="dense gradients"):
        tt.TrainStep(model, loss, opt, max_grad_norm=1.0)
    opt.release_tables()
    tt.TrainStep(model, loss, opt, max_grad_norm=1.0)
    with pytest.raises(ValueError, match="must not be negative"):
        tt.TrainStep(model, loss, opt, max_grad_norm=-1.0)


def test_train_step_hands_each_batch_its_own_loss_inputs():
    torch.manual_seed(4)
    model = _Linear()
    seen = []

    def loss_fn(a, b, target=None, mask=None):
        seen.append((target, mask))
        return ((a - b) * (1.0 if target is None else target)).square().mean()

    step = tt.TrainStep(model, loss_fn, torch.optim.SGD(model.parameters(), lr=0.1))
    x, y, t1, t2 = torch.randn(4, 6), torch.randn(4, 5), torch.rand(4, 5), torch.rand(4, 5)
    step(x, y, target=t1)
    step(x, y, target=t2, mask=None)
    step(x, y)
    assert seen[0][0] is t1 and seen[1][0] is t2
    assert seen[2] == (None, None) and seen[1][1] is None
    with pytest.raises(TypeError, match="loss input target must be a tensor"):
        step(x, y, target=0.5)


def test_a_live_graph_of_a_parameter_is_found():
    a, b = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3))
    assert _lib.nodes().live_leaf([a, b]) == -1
    loss = (b * 2).sum()
    assert _lib.nodes().live_leaf([a, b]) == 1
    loss.backward()
    assert _lib.nodes().live_leaf([a, b]) == 1  # (its tensors are freed, its nodes are not)
    loss = loss.detach()
    assert _lib.nodes().live_leaf([a, b]) == -1


def test_a_table_differentiated_both_ways_is_refused():
    d, grad = ops.DeferredTableGrad(), torch.zeros(2, 2)
    d.added_dense()
    assert not d.pending(grad)  # a dense gradient alone is stepped as usual ...
    d.parts.append(("part",))
    assert d.pending(grad)  # ... and says nothing about the next step
    d.added_dense()
    assert d.pending(None)  # dropped by zero_grad before the step
    d.added_dense()
    with pytest.raises(RuntimeError, match="pooled lookups only"):
        d.pending(grad)
    assert not d.parts and not d.pending(grad)


@pytest.mark.parametrize("make, err, msg", [
    (lambda: ops.Int4Rows.quantize(torch.zeros(4)), ValueError, "x must be"),
    (lambda: ops.Int4Rows.quantize(torch.zeros(4, 8), group=48), ValueError, "group must be"),
    (lambda: ops.Int4Rows.quantize(torch.zeros(4, 4097)), ValueError, "rows of 1 to 4096"),
    (lambda: ops.Int4Rows.quantize(torch.zeros(4, 8, dtype=torch.int32)), TypeError, "x must be float32"),
    (lambda: ops.Int4Rows.quantize(torch.zeros(4, 8)), RuntimeError, "no CPU fallback"),
    (lambda: ops.Int4Rows.from_codes(torch.zeros(4, 40), torch.zeros(4, 2).bfloat16()), ValueError, "int8"),
    (lambda: ops.Int4Rows.from_codes(torch.zeros(4, 40, dtype=torch.int8), torch.zeros(4, 1).bfloat16()), ValueError,
     r"scales must be \(4, 2\)"),
    (lambda: ops.Int4Rows.from_codes(torch.zeros(4, 40, dtype=torch.int8), torch.zeros(4, 2)), ValueError, "bfloat16"),
    (lambda: ops.Int4Rows(torch.zeros(7, dtype=torch.uint8), torch.zeros(7, dtype=torch.uint8), 4, 40, 32), ValueError,
     "codes must be 512"),
])
def test_int4_refusals(make, err, msg):
    with pytest.raises(err, match=msg):
        make()


def test_scores_without_a_gradient_are_not_differentiated_silently(monkeypatch):
    """The scores of queries that need a gradient are computed, and refused where they are differentiated."""
    from torch.autograd import forward_ad

    monkeypatch.setattr(ops, "_int4_scores", lambda q, rows: q.detach() @ rows.t())
    q, rows = torch.randn(3, 8, requires_grad=True), torch.randn(5, 8)
    scores = ops.int4_scores(q, rows)
    assert torch.equal(scores, q @ rows.t())
    with pytest.raises(RuntimeError, match="int4_scores has no gradient"):
        scores.sum().backward()
    with torch.no_grad():
        assert not ops.int4_scores(q, rows).requires_grad
    assert not ops.int4_scores(q.detach(), rows).requires_grad
    with forward_ad.dual_level():
        assert torch.equal(ops.int4_scores(q.detach(), rows), scores)
        with pytest.raises(RuntimeError, match="int4_scores has no derivative"):
            ops.int4_scores(forward_ad.make_dual(q.detach(), torch.ones(3, 8)), rows)


def test_search_refuses_an_unknown_index_type():
    with pytest.raises(ValueError, match="index_dtype"):
        tt.search.TwoTowerSearch(torch.nn.Identity(), device="cpu", index_dtype="int8")


def test_lookup_embedding_on_the_cpu_is_the_plain_gather():
    emb = tt.embeddings.build("lookup", vocab_size=9, embedding_dim=6, scale=2.0)
    ids = torch.tensor([[1, 0, 8]])
    assert torch.equal(emb(ids), emb.embedding(ids) * 2.0)
    assert list(emb.state_dict()) == ["embedding.weight"]


class _Pooler(torch.nn.Module):
    def __init__(self, embedding):
        super().__init__()
        self.embedding = embedding

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return self.embedding(ids).sum(1)


@pytest.mark.parametrize("scale", [1.0, 2.0])
@pytest.mark.parametrize("how", [torch.fx.symbolic_trace, torch.jit.script,
                                 lambda m: torch.jit.trace(m, torch.tensor([[1, 2]])),
                                 lambda m: torch.compile(m, backend="eager", fullgraph=True),
                                 lambda m: torch.export.export(m, (torch.tensor([[1, 0, 8]]),)).module()],
                         ids=["fx", "script", "trace", "compile", "export"])
def test_lookup_embedding_can_be_traced_and_compiled(how, scale):
    emb = tt.embeddings.build("lookup", vocab_size=9, embedding_dim=6, scale=scale)
    ids = torch.tensor([[1, 0, 8]])
    for module in (emb, _Pooler(emb)):
        got = how(module)(ids)
        assert torch.equal(got, module(ids))
        want = torch.autograd.grad(module(ids).square().sum(), emb.weight)[0]
        assert torch.equal(torch.autograd.grad(got.square().sum(), emb.weight)[0], want)


def test_lookup_embedding_pickled_without_a_scale():
    import copy

    emb = tt.embeddings.build("lookup", vocab_size=9, embedding_dim=6)
    old = copy.deepcopy(emb)
    del old.__dict__["scale"]
    ids = torch.tensor([[1, 0, 8]])
    assert torch.equal(old(ids), emb(ids))


def test_only_an_embedding_as_torch_made_it_is_plain(monkeypatch):
    """What a user puts around the inner embedding's forward must run: its own hooks, global ones, another forward."""
    from twotower_amd import embeddings

    def fresh():
        return torch.nn.Embedding(5, 4, padding_idx=0)

    assert embeddings._plain_embedding(fresh())
    m = fresh()
    m.forward = lambda ids: torch.zeros(1)
    assert not embeddings._plain_embedding(m)
    handles = [lambda: torch.nn.modules.module.register_module_forward_hook(lambda *a: None),
               lambda: torch.nn.modules.module.register_module_forward_pre_hook(lambda *a: None),
               lambda: torch.nn.modules.module.register_module_full_backward_hook(lambda *a: None),
               lambda: torch.nn.modules.module.register_module_full_backward_pre_hook(lambda *a: None)]
    for register in handles:
        handle = register()
        try:
            assert not embeddings._plain_embedding(fresh())
        finally:
            handle.remove()
    assert embeddings._plain_embedding(fresh())
    monkeypatch.setattr(torch.nn.Embedding, "forward", lambda self, ids: None)
    assert not embeddings._plain_embedding(fresh())


def test_function_modes_observe_the_lookup():
    from twotower_amd import embeddings

    class Mode(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    assert not embeddings._observed()
    with Mode():
        assert embeddings._observed()
    with torch.device("cpu"):  # factories' default: nothing that follows a lookup
        assert not embeddings._observed()


def _dp_clip_worker(rank, port, q):
    import os

    import torch.distributed as dist

    from twotower_amd import train_step

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        train_step.clip_grad_norm_ = torch.nn.utils.clip_grad_norm_  # (the kernels need a GPU; the order is what is tested)
        model, step, batch = _dp_clip_step()
        step(*(t[rank * 4:(rank + 1) * 4] for t in batch))
        q.put((rank, [p.detach().numpy() for p in model.parameters()], float(step.grad_norm)))
    finally:
        dist.destroy_process_group()


class _Linear(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = torch.nn.Linear(6, 5)

    def forward(self, q, p):
        return self.lin(q), p


def _dp_clip_step():
    torch.manual_seed(3)
    model = _Linear().double()
    opt = torch.optim.SGD(model.parameters(), lr=1.0)
    batch = torch.randn(8, 6, dtype=torch.float64), torch.randn(8, 5, dtype=torch.float64)
    return model, tt.TrainStep(model, lambda a, b: ((a - b) ** 2).mean(), opt, max_grad_norm=0.1), batch


def test_data_parallel_clipping_uses_the_global_gradient():
    """Two ranks, half the batch each: the all-reduced gradient is clipped (by one norm on both ranks), so the
    step equals the single-process step on the whole batch."""
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = torch.multiprocessing.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_dp_clip_worker, args=(r, port, q)) for r in range(2)]
    [p.start() for p in procs]
    got = dict((r, (ps, n)) for r, ps, n in (q.get(timeout=120) for _ in range(2)))
    [p.join(60) for p in procs]
    model, step, (x, y) = _dp_clip_step()
    loss = ((model.lin(x) - y) ** 2).mean()
    loss.backward()
    norm = torch.nn.utils.clip_grad_norm_(model.parameters(), 0.1).item()
    assert norm > 0.1
    with torch.no_grad():
        want = [p - p.grad for p in model.parameters()]
    for ps, n in got.values():
        assert abs(n - norm) < 1e-12
        for a, b in zip(ps, want):
            assert abs(torch.from_numpy(a) - b).max() < 1e-12


def test_a_capture_waits_for_the_watchdogs_of_gpu_groups(monkeypatch):
    """Only groups whose watchdog queries events are waited for (gloo has none), and none without a group."""
    from twotower_amd import distributed

    waited = []

    class Group:
        def __init__(self, kind):
            self.kind = kind

        def _wait_for_pending_works(self):
            waited.append(self.kind)

    distributed.settle_watchdogs()  # no process group
    monkeypatch.setattr(distributed, "_backend_kind", lambda g: g.kind)
    distributed.settle_watchdogs([Group("gloo"), Group("nccl"), Group("other"), Group("nccl")])
    assert waited == ["nccl", "nccl"]
    assert hasattr(torch.distributed.ProcessGroup, "_wait_for_pending_works")


class _Halved(torch.autograd.Function):
    """A view whose gradient is scaled (gradient scaling or reversal layers have this form)."""

    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        return g * 0.5


def _buffer_node(seen=None):
    """A loss of consecutive blocks whose gradients are blocks of one buffer (as preference_loss's are)."""

    class Node(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *blocks):
            ctx.save_for_backward(*blocks)
            return sum((b ** 2).sum() for b in blocks)

        @staticmethod
        def backward(ctx, g):
            whole = 2 * g * torch.cat([b.reshape(-1, b.shape[-1]) for b in ctx.saved_tensors])
            if seen is not None:
                seen.append(whole)
            out, at = [], 0
            for b in ctx.saved_tensors:
                rows = b.numel() // b.shape[-1]
                out.append(whole[at:at + rows].view(b.shape))
                at += rows
            return tuple(out)

    return Node.apply


def _split_case(sizes=(3, 3, 6)):
    x = torch.randn(sum(sizes), 4, dtype=torch.float64, requires_grad=True)
    y = x * 1.0
    return x, y, _lib.nodes().split_rows(y, list(sizes))


def test_split_rows_is_torch_split():
    x, y, blocks = _split_case((3, 0, 6))
    assert [b.shape[0] for b in blocks] == [3, 0, 6] and all(b._base is y for b in blocks)
    assert all(torch.equal(a, b) for a, b in zip(blocks, torch.split(y, [3, 0, 6])))
    with pytest.raises(RuntimeError, match="inplace"):  # as torch.split's outputs
        blocks[0].mul_(2)
    (g,) = torch.autograd.grad((blocks[2] ** 3).sum(), x, create_graph=True)  # blocks without a gradient count zeros
    assert torch.equal(g, torch.cat([torch.zeros(3, 4), 3 * x[3:] ** 2]))
    (h,) = torch.autograd.grad(g.sum(), x)
    assert torch.equal(h, torch.cat([torch.zeros(3, 4), 6 * x[3:]]))
    for sizes in ([3, 4], [], [-1, 10], [10]):
        with pytest.raises(ValueError, match="split_rows"):
            _lib.nodes().split_rows(y, sizes)
    assert torch.autograd.gradcheck(lambda t: _lib.nodes().split_rows(t, [2, 1]), torch.randn(3, 2, dtype=torch.float64,
                                                                                             requires_grad=True))


def test_split_rows_hands_one_buffer_on_without_a_copy():
    seen = []
    x, y, (a, b, c) = _split_case()
    got = []
    y.register_hook(lambda g: got.append((g.data_ptr(), torch.equal(g, 2 * y))))
    _buffer_node(seen)(a, b, c.view(3, 2, 4)).backward()
    assert got == [(seen[0].data_ptr(), True)]
    x, y, (a, b, c) = _split_case()  # another order is joined
    (g,) = torch.autograd.grad(_buffer_node()(b, a, c), y)
    assert torch.equal(g, 2 * y)


@pytest.mark.parametrize("sizes", [(1, 1, 2), (1, 0, 3), (0, 2, 1), (1,), (2, 1)])
def test_split_rows_of_short_blocks(sizes):
    x, y, blocks = _split_case(sizes)
    (g,) = torch.autograd.grad(_buffer_node()(*blocks), y)
    assert torch.equal(g, 2 * y) and g.shape == y.shape
    whole = torch.randn(sum(sizes), 4, dtype=torch.float64)  # one row's stride means nothing
    parts = [w.as_strided(w.shape, (77, 1), w.storage_offset()) if len(w) == 1 else w for w in whole.split(list(sizes))]
    assert torch.equal(torch.autograd.grad(_lib.nodes().split_rows(x * 1.0, list(sizes)), x, parts)[0], whole)


def test_split_rows_blocks_keep_what_autograd_has_on_them():
    """Functions, hooks, retained gradients and other uses of a block, and gradients with respect to the blocks."""
    node = _buffer_node()
    x, y, (a, b, c) = _split_case()
    (g,) = torch.autograd.grad(node(_Halved.apply(a), b, c), x)
    assert torch.equal(g, torch.cat([x[:3], 2 * x[3:]]))
    x, y, (a, b, c) = _split_case()
    b.register_hook(lambda g: g * 3)
    a.retain_grad()
    node(a, b, c).backward()
    assert torch.equal(x.grad, torch.cat([2 * x[:3], 6 * x[3:6], 2 * x[6:]])) and torch.equal(a.grad, 2 * a)
    x, y, blocks = _split_case()
    assert all(torch.equal(g, 2 * t) for g, t in zip(torch.autograd.grad(node(*blocks), blocks), blocks))
    x, y, (a, b, c) = _split_case()
    (g,) = torch.autograd.grad(node(a, b, c) + (5 * b).sum(), x)
    assert torch.equal(g, torch.cat([2 * x[:3], 2 * x[3:6] + 5, 2 * x[6:]]))


def _split_rows(y, sizes):
    return _lib.nodes().split_rows(y, sizes)


def _base_and_blocks(split=torch.split):
    y = torch.randn(12, 4, requires_grad=True) * 1.0
    return y, list(split(y, [3, 3, 6]))


@pytest.mark.parametrize("split", [torch.split, _split_rows, lambda y, s: (y[:3], y.narrow(0, 3, 3), y[6:])])
def test_losses_take_the_base_only_where_it_stands_for_its_views(split):
    """The losses that differentiate the common tensor of q, p and n: whatever autograd has on a view must not be
    passed by."""
    y, (q, p, n) = _base_and_blocks(split)
    assert losses._direct(y, q, p, n.view(3, 2, 4), rows=True) == (split is _split_rows)
    assert losses._packed(q, p, n) is y and losses._packed(q, p, n.view(3, 2, 4).view(6, 4)) is y
    assert losses._candidates(p, n)._base is y
    assert losses._packed(_Halved.apply(q), p, n) is None
    assert losses._packed(q, p, _Halved.apply(n)) is None
    assert losses._candidates(_Halved.apply(p), n)._base is None
    p.register_hook(lambda g: g * 2)
    assert losses._packed(q, p, n) is None and losses._candidates(p, n)._base is None
    y, (q, p, n) = _base_and_blocks(split)
    n.retain_grad()
    assert losses._packed(q, p, n) is None and losses._candidates(p, n)._base is None
    y, (q, p, n) = _base_and_blocks(split)
    m = n.view(3, 2, 4)
    m.register_hook(lambda g: None)
    assert losses._packed(q, p, m.view(6, 4)) is None
    with torch.no_grad():
        assert losses._packed(y[:3], p, n) is None and losses._candidates(y[3:6], n)._base is None
        assert losses._packed(*(t.detach() for t in (q, p, n))) is None  # (the base still needs its gradient)
    x = torch.randn(12, 4)
    q, p, n = split(x, [3, 3, 6])
    assert losses._packed(q, p, n) is x  # no gradient anywhere
    assert losses._packed(q.requires_grad_(True), p, n) is None


def test_candidates_keep_what_autograd_has_on_them():
    y, (q, p, n) = _base_and_blocks()
    out = losses._candidates(p, n)
    (want,) = torch.autograd.grad((out * torch.arange(9.0)[:, None]).sum(), y, retain_graph=True)
    out = losses._candidates(_Halved.apply(p), n)
    (got,) = torch.autograd.grad((out * torch.arange(9.0)[:, None]).sum(), y)
    assert torch.equal(got[3:6], 0.5 * want[3:6]) and torch.equal(got[6:], want[6:])


def _make(*args):
    import os
    import subprocess

    where = os.path.join(os.path.dirname(os.path.abspath(tt.__file__)), "csrc")
    return subprocess.run(["make", "-C", where, *args], check=True, capture_output=True, text=True).stdout


def test_the_library_builds_without_torch():
    assert "nodes.cpp" in _make("-n", "-B")
    for how in (["TORCH="], ["PYINC=/nowhere"], ["TORCH=/nowhere"], ["PYTHON=/nowhere/python"], ["lib"]):
        plan = _make("-n", "-B", *how)
        assert "lookup.hip" in plan and "nodes.cpp" not in plan
        assert ("needs _nodes.so" in plan) == (how != ["lib"])


def test_the_module_is_built_anew_for_another_torch(tmp_path):
    """A compiler that only notes its runs: a second make does nothing, one with another torch compiles."""
    import sys

    stub, log = tmp_path / "cxx.py", tmp_path / "log"
    stub.write_text(f"import sys; open(sys.argv[sys.argv.index('-o') + 1], 'w'); open({str(log)!r}, 'a').write('x')")
    torches = []
    for version in ("1", "2"):
        root = tmp_path / version
        (root / "include" / "torch").mkdir(parents=True)
        (root / "include" / "torch" / "extension.h").touch()
        (root / "version.py").write_text(f"__version__ = '{version}'")
        torches.append(root)
    (tmp_path / "Python.h").touch()
    for root, runs in ((torches[0], 1), (torches[0], 1), (torches[1], 2), (torches[1], 2), (torches[0], 3)):
        out = tmp_path / "_nodes.so"
        _make(str(out), f"NODES={out}", f"BUILD={tmp_path}/build", f"CXX={sys.executable} {stub}", f"TORCH={root}",
              f"PYINC={tmp_path}")
        assert len(log.read_text()) == runs


# ---------------------------------------------------------------------------------------------
# C ABI


def _clip(src=P, dst=P, n=3, st=0, dt=0, max_norm=1.0, ws=1 << 20):
    a = [(ctypes.c_int64 * 1)(v or 0) for v in (src, dst, n)]
    return (*a, bytes([st]), bytes([dt]), 1, 0, max_norm, 1, P, P, ws, None)


@pytest.mark.parametrize("name, args, msg", [
    ("tt_lookup_fwd", (P, 0, 0, 4, 4, P, 0, 1, 1.0, P, 0, None), "V=0 out of range"),
    ("tt_lookup_fwd", (P, 0, 5, 0, 4, P, 0, 1, 1.0, P, 0, None), "E=0"),
    ("tt_lookup_fwd", (P, 0, 5, 4, 3, P, 0, 1, 1.0, P, 0, None), "ld_table=3"),
    ("tt_lookup_fwd", (P, 0, 5, 4, 4, None, 0, 1, 1.0, P, 0, None), "ids is NULL"),
    ("tt_lookup_fwd", (P, 0, 5, 4, 4, P, 2, 1, 1.0, P, 0, None), "ids_dtype=2"),
    ("tt_lookup_fwd", (P, 1, 5, 4, 4, P, 0, 1, 1.0, P, 0, None), "rows of type 0"),
    ("tt_lookup_fwd", (P, 0, 5, 4, 4, P, 6, 1, 1.0, P, 0, None), "ids_dtype=2"),
    ("tt_lookup_bwd", (P, 0, P, 4, 1, 5, 4, -1, 1.0, P, 0, None, 0, None, 0, None), "ids_dtype=4"),
    ("tt_lookup_fwd", (P, 0, 5, 4, 4, P, 0, 2 ** 31, 1.0, P, 0, None), "out of range"),
    ("tt_lookup_fwd", (None, 0, 5, 4, 4, P, 0, 1, 1.0, P, 0, None), "null pointer"),
    ("tt_lookup_bwd", (None, 0, P, 0, 1, 5, 4, -1, 1.0, P, 0, None, 0, None, 0, None), "null pointer"),
    ("tt_lookup_bwd", (P, 0, P, 0, 9000, 5, 4, -1, 1.0, P, 0, None, 0, P, 1 << 30, None), "plan too small"),
    ("tt_lookup_bwd", (P, 0, P, 0, 9000, 5, 4, -1, 1.0, P, 0, P, 1 << 30, P, 8, None), "workspace too small"),
    ("tt_lookup_plan", (P, 0, 9000, 5, -1, P, 100, None), "workspace too small"),
    ("tt_lookup_plan", (None, 0, 9000, 5, -1, P, 1 << 30, None), "ids is NULL"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 3, 2, 1, 4, None, None, 0, 1.0, 1.0, 0.0, P, None, P, P, P, 16, None),
     "element type 3"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 0, 2, 0, 4, None, None, 0, 1.0, 1.0, 0.0, P, None, P, P, P, 16, None),
     "bad shape"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 0, 2, 1, 4, None, None, 2, 1.0, 1.0, 0.0, P, None, P, P, P, 16, None),
     "loss kind 2"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 0, 2, 1, 4, None, None, 0, 0.0, 1.0, 0.0, P, None, P, P, P, 16, None),
     "must be positive"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 0, 2, 1, 4, None, None, 0, 1.0, 1.0, 0.0, P, None, P, P, P, 15, None),
     "workspace too small"),
    ("tt_preference_fwd", (P, 4, P, 4, P, 4, 4, 0, 2, 1, 4, None, None, 0, 1.0, 1.0, 0.0, P, None, P, None, P, 16, None),
     "null pointer"),
    ("tt_preference_bwd", (P, 4, P, 4, P, 4, 4, 0, 2, 1, 4, None, 1.0, P, P, None, P, P, P, None), "null pointer"),
    ("tt_clip_grads", (None, None, None, None, None, 1, 0, 1.0, 1, P, P, 1 << 20, None), "null pointer"),
    ("tt_clip_grads", _clip(max_norm=-1.0), "max_norm"),
    ("tt_clip_grads", _clip(ws=8), "workspace too small"),
    ("tt_clip_grads", _clip(dst=None), "tensor 0 is NULL"),
    ("tt_clip_grads", _clip(dt=1), "of type 0 into type 1"),
    ("tt_clip_grads", _clip(st=3, dt=3), "of type 3 into type 3"),
    ("tt_clip_grads", _clip(n=-1), "-1 elements"),
    ("tt_int4_quantize", (P, 0, 4, 4097, 4097, 32, P, P, None), "H=4097"),
    ("tt_int4_quantize", (P, 0, 4, 64, 63, 32, P, P, None), "ld=63"),
    ("tt_int4_quantize", (P, 0, 4, 64, 64, 16, P, P, None), "group=16"),
    ("tt_int4_quantize", (P, 0, 4, 64, 64, 32, P + 4, P, None), "16-byte aligned"),
    ("tt_int4_pack", (None, P, 4, 64, 32, P, P, None), "null pointer"),
    ("tt_int4_unpack", (P, P, 4, 64, 32, None, None), "null pointer"),
    ("tt_int4_scores", (P, 0, 1, 63, P, P, 4, 64, 32, P, None), "ldq=63"),
    ("tt_int4_scores", (P, 7, 1, 64, P, P, 4, 64, 32, P, None), "query type 7"),
    ("tt_int4_scores", (P, 0, 1, 64, None, P, 4, 64, 32, P, None), "null pointer"),
])
def test_c_abi_refusals(name, args, msg):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc == -1
    assert msg in _lib.last_error(), _lib.last_error()


def test_c_abi_sizes():
    lib = _lib.lib()
    for n, short in ((_lib.TT_LOOKUP_DIRECT_TOKENS, True), (_lib.TT_LOOKUP_DIRECT_TOKENS + 1, False)):
        for rows, E, dtype in ((n, 256, 0), (n, 512, 1), (n // 2 + (n & 1), 260, 0), (n // 4 + (n & 1), 2048, 2),
                               (n // 2 + (n & 1), 339, 1)):
            sizes = lib.tt_lookup_plan_size(rows, 50, E, dtype), lib.tt_lookup_bwd_ws_size(rows, E, dtype)
            assert [s == 0 for s in sizes] == [short, short]  # short calls take neither
    assert lib.tt_lookup_bwd_ws_size(100_000, 8, 0) == (2 * 3125 + 97) * 8 * 4  # heads, tails, super-tiles
    assert lib.tt_lookup_plan_size(100_000, 50, 8, 0) > 4 * 4 * 100_000
    assert lib.tt_int4_codes_bytes(17, 33) == 2 * 2 * 256  # two tiles of 16 rows, two 32-column blocks
    assert lib.tt_int4_scales_bytes(17, 33, 32) == 2 * 1 * 16 * 4 * 2
    assert lib.tt_clip_ws_size(1) == lib.tt_clip_ws_size(1000) == 2048 * 8


# ---------------------------------------------------------------------------------------------
# the formulas the kernels' gradients are tested with, against central differences in 64 bits
def pair_terms(h, beta, smooth, kind):
    """(loss, d loss / d h) of margins in 64 bits (numerically stable, from the definition)."""
    if kind == "sigmoid":
        sp = torch.nn.functional.softplus
        x = beta * h
        return (1 - smooth) * sp(-x) + smooth * sp(x), beta * (smooth - torch.sigmoid(-x))
    return (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)


@pytest.mark.parametrize("kind, smooth", [("sigmoid", 0.0), ("sigmoid", 0.1), ("squared", 0.0)])
def test_pair_derivative_against_differences(kind, smooth):
    h = torch.linspace(-6, 6, 41, dtype=torch.float64)
    step = 1e-5  # a central difference is off by step^2 l''' / 6 + 2^-53 |l| / step < 1e-9
    lo, hi = (pair_terms(h + d, 0.7, smooth, kind)[0] for d in (-step, step))
    _, dl = pair_terms(h, 0.7, smooth, kind)
    assert (((hi - lo) / (2 * step)) - dl).abs().max() < 1e-8
