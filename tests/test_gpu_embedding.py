"""Embedding of tokens and the gradients of its tables, against 64 bits: every value is at most one rounding to its type and the roundings of
its fp32 sum away; the same bits in every run."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# tokens, rows, columns: one and few, sizes around packs, warps, stretches and passes of the sort, several stretches per row
SIZES = [(1, 1, 1), (1, 50257, 1024), (2, 7, 8), (15, 255, 33), (16, 256, 64), (17, 257, 40), (129, 5, 1027), (300, 65535, 24), (1000, 65536, 17), (4099, 3, 128),
         (8192, 50257, 256), (70001, 1000, 48)]


def table(rows, cols, dtype, gen):
    return torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)


def check(got, want, magnitude, terms):
    """One rounding to the type (half a step, eps / 2 of the value; in fp16 at least half of the smallest step, 2**-25), and one to fp32 per term."""
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2 ** -8) + magnitude * terms * 2.0 ** -23 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert bool(((got.double() - want).abs() <= tol).all())


def summed(index, g, rows):
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64, device="cuda")
    return out.index_add_(0, index.long(), g.double())


def gradients(ids, w, pos, p, scale, pad, g):
    keep = torch.ones_like(ids, dtype=torch.float64) if pad is None else (ids != pad).double()
    gs = g.double() * keep[:, None] * scale
    want = [(summed(ids, gs, w.shape[0]), summed(ids, gs.abs(), w.shape[0]))]
    if pos is not None:
        want.append((summed(pos, g, p.shape[0]), summed(pos, g.abs(), p.shape[0])))
    return want


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("with_positions", [False, True])
def test_forward_and_gradients(n, v, d, dtype, with_positions):
    from dfccl_b200.ops.embedding import embedding
    gen = torch.Generator(device="cuda").manual_seed(n + v + d)
    w = table(v, d, dtype, gen).requires_grad_(True)
    ids = (torch.rand(n, generator=gen, device="cuda") ** 3 * v).long().clamp_(max=v - 1)
    scale, pad = (1.0, None) if with_positions else (1.7, int(ids[0]))
    pos = p = None
    if with_positions:
        p = table(37, d, dtype, gen).requires_grad_(True)
        pos = (torch.arange(n, device="cuda") * 5 % 37).int()
    out = embedding(ids, w, scale=scale, positions=pos, position_weight=p, padding_idx=pad)
    want = w.detach().double()[ids] * scale + (p.detach().double()[pos.long()] if pos is not None else 0.0)
    assert out.shape == (n, d) and out.dtype == dtype
    check(out.detach(), want, want.abs() + (w.detach().double()[ids] * scale).abs(), 2)
    g = torch.randn(n, d, generator=gen, device="cuda").to(dtype)
    if dtype == torch.float16:
        g = g / 64
    tables = [w] + ([p] if p is not None else [])
    got = torch.autograd.grad(out, tables, g, retain_graph=True)
    for x, (value, size) in zip(got, gradients(ids, w, pos, p, scale, pad, g)):
        check(x, value, size, n + 1)
    again = torch.autograd.grad(out, tables, g)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("n", [16, 17, 2048, 140000])
@pytest.mark.parametrize("kind", ["one", "two", "rising", "falling"])
def test_orders_of_tokens(n, kind):
    """All tokens alike (one row that goes through every stretch), two rows, rising and falling ids."""
    from dfccl_b200.ops.embedding import embedding
    v, d = 40000, 16
    at = torch.arange(n, device="cuda")
    ids = {"one": at * 0 + 255, "two": at % 2 * 39999, "rising": at % v, "falling": v - 1 - at % v}[kind]
    w = torch.zeros(v, d, device="cuda", requires_grad=True)
    g = torch.randn(n, d, device="cuda")
    got, = torch.autograd.grad(embedding(ids, w), [w], g)
    check(got, summed(ids, g, v), summed(ids, g.abs(), v), n)


def test_tokens_in_their_order():
    """The fp32 sum of a row runs over its tokens in their order: within a stretch of 16 it is the running sum, bit by bit."""
    from dfccl_b200.ops.embedding import embedding
    gen = torch.Generator(device="cuda").manual_seed(3)
    n, d = 16, 64
    ids = torch.tensor([5, 900, 5, 5, 0, 900, 5, 70000, 5, 0, 5, 5, 900, 5, 5, 5], device="cuda")
    w = torch.zeros(70001, d, device="cuda", requires_grad=True)
    g = torch.randn(n, d, generator=gen, device="cuda") * torch.logspace(-3, 3, n, device="cuda")[:, None]
    got, = torch.autograd.grad(embedding(ids, w), [w], g)
    for v in (0, 5, 900, 70000):
        run = torch.zeros(d, device="cuda")
        for i in (ids == v).nonzero()[:, 0].tolist():
            run = run + g[i]
        assert torch.equal(got[v], run)


def test_tokens_outside_the_tables():
    """Rows of NaN, no gradient, and nothing else touched."""
    from dfccl_b200.ops.embedding import embedding
    ids = torch.tensor([[3, -1, 9], [10, 2 ** 40, 0]], device="cuda")
    pos = torch.tensor([[0, 1, 4], [2, 3, -5]], device="cuda")
    w, p = torch.ones(10, 24, device="cuda", requires_grad=True), torch.ones(4, 24, device="cuda", requires_grad=True)
    out = embedding(ids, w, positions=pos, position_weight=p)
    bad = torch.tensor([[False, True, True], [True, True, True]], device="cuda")
    assert bool((out.isnan() == bad[..., None]).all()) and bool((out[0, 0] == 2.0).all())
    gw, gp = torch.autograd.grad(out, [w, p], torch.ones_like(out))
    assert gw[:, 0].tolist() == [1.0, 0, 0, 1.0, 0, 0, 0, 0, 0, 1.0] and gp[:, 0].tolist() == [1.0, 1.0, 1.0, 1.0]


def test_strides_and_shapes():
    """Tables that are slices or transposed, ids that are every other of a matrix, no tokens at all, gradients that are a broadcast value."""
    from dfccl_b200.ops.embedding import embedding
    gen = torch.Generator(device="cuda").manual_seed(7)
    wide = torch.randn(50, 100, generator=gen, device="cuda")
    for w in (wide[:, 3:67], wide[:, 4:68], wide.t(), wide[::2], wide[:1].expand(50, 100)):
        w = w.detach().requires_grad_(True)
        ids = torch.randint(0, w.shape[0], (6, 10), generator=gen, device="cuda")[:, ::2].t()
        out = embedding(ids, w)
        assert torch.equal(out, w[ids]) and out.shape == (5, 6, w.shape[1])
        out.sum().backward()
        assert torch.equal(w.grad[:, 0], torch.bincount(ids.reshape(-1), minlength=w.shape[0]).float())
    w = wide.detach().requires_grad_(True)
    none = embedding(torch.empty(0, 4, dtype=torch.int64, device="cuda"), w)
    assert none.shape == (0, 4, 100)
    none.sum().backward()
    assert bool((w.grad == 0).all())


def test_a_table_of_one_row_with_any_stride():
    from dfccl_b200.ops.embedding import embedding
    one = torch.arange(40.0, device="cuda").as_strided((1, 40), (0, 1))
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    assert torch.equal(embedding(ids, one, positions=ids, position_weight=one), 2 * one.expand(3, 40))


def test_tables_and_results_of_more_elements_than_31_bits_count():
    from dfccl_b200.ops.embedding import embedding
    rows, d = 530003, 4096
    gen = torch.Generator(device="cuda").manual_seed(13)
    small = torch.randn(100, d, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_(True)
    ids = torch.randint(0, 100, (rows,), generator=gen, device="cuda")
    out = embedding(ids, small)
    assert torch.equal(out[-1000:], small[ids[-1000:]])
    g = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    g[-1000:] = 1
    assert torch.equal(torch.autograd.grad(out, [small], g)[0][:, 7].float(), torch.bincount(ids[-1000:], minlength=100).float())
    del out
    large = g.requires_grad_(True)                            # its last rows are ones, the others zeros
    ids = torch.tensor([rows - 1, 0, rows - 2, rows - 1, rows - 1001], device="cuda")
    out = embedding(ids, large)
    assert out[:, -1].tolist() == [1.0, 0.0, 1.0, 1.0, 0.0]
    grad = torch.autograd.grad(out, [large], torch.ones_like(out))[0]
    assert grad[[0, 1, rows - 1001, rows - 2, rows - 1], -1].tolist() == [1.0, 0.0, 1.0, 1.0, 2.0] and grad.sum(dtype=torch.float64).item() == 5.0 * d


def test_other_stream_and_graph():
    """On a stream of its own; forward and backward captured and replayed for other tokens, beside a second graph."""
    from dfccl_b200.ops.embedding import embedding
    gen = torch.Generator(device="cuda").manual_seed(11)
    w = torch.randn(3001, 72, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_(True)
    g = torch.randn(777, 72, generator=gen, device="cuda").to(torch.bfloat16)
    batches = [torch.randint(0, 3001, (777,), generator=gen, device="cuda") for _ in range(3)]

    def step(ids):
        out = embedding(ids, w, scale=0.5)
        return out.detach(), torch.autograd.grad(out, [w], g)[0]

    want = [step(b) for b in batches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(batches[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for _ in range(2):
        ids = batches[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(ids)
        graphs.append((ids, graph, out))
    for turn in range(3):
        for k, (ids, graph, _) in enumerate(graphs):
            ids.copy_(batches[(turn + k) % 3])
            graph.replay()
        for k, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(turn + k) % 3]))


@pytest.mark.parametrize("end", ["wte", "wpe"])
@pytest.mark.parametrize("option", ["padding_idx", "max_norm", "scale_grad_by_freq", "sparse", "dtype"])
def test_a_stage_respects_its_embeddings_options(option, end):
    """A table that does more than look up keeps doing it where the stage's ends are fused."""
    from dfccl_b200 import native as nv
    from dfccl_b200.models.gpt2 import GPT2Config, GPT2Stage
    from dfccl_b200.ops.fused_linear import TpGroup
    (comm,) = nv.Comm.init_loopback(1, torch.cuda.current_device())
    cfg = GPT2Config(n_layer=2, d_model=256, n_head=4, seq_len=128, vocab=300)
    tp = TpGroup(comm, None, torch.device("cuda", torch.cuda.current_device()))
    tokens = torch.randint(0, 40, (4, 129), device="cuda")
    tokens[0, 0] = 7
    results = []
    for fused in (False, True):
        stage = GPT2Stage(cfg, tp, 0, 2, 4, fused_ends=fused)
        old = getattr(stage, end)
        kind = {"padding_idx": {"padding_idx": 7}, "max_norm": {"max_norm": 0.125}, "scale_grad_by_freq": {"scale_grad_by_freq": True}, "sparse": {"sparse": True}}.get(option, {})
        new = torch.nn.Embedding(old.num_embeddings, old.embedding_dim, device="cuda", dtype=torch.float32 if option == "dtype" else torch.bfloat16, **kind)
        with torch.no_grad():
            new.weight.copy_(old.weight)
        setattr(stage, end, new)
        stage.blocks = torch.nn.ModuleList()                 # what the first stage hands on is the embedding
        h = stage(tokens[:, :-1])
        assert not stage.ran_fused_ends
        grad = torch.linspace(-1, 1, h.numel(), device="cuda").view_as(h).to(h.dtype)
        grads = torch.autograd.grad(h, [stage.wte.weight, stage.wpe.weight], grad)
        results.append([h.detach(), new.weight.detach().clone()] + [g.double() if not g.is_sparse else torch.zeros(g.shape, dtype=torch.float64, device="cuda").index_add_(
            0, g._indices()[0], g._values().double()) for g in grads])
    comm.destroy()
    (h0, w0, *g0), (h1, w1, *g1) = results
    assert h0.dtype == h1.dtype and torch.equal(h0, h1) and torch.equal(w0, w1)
    for a, b in zip(g0, g1):                                 # (sums in another order, rounded once: bf16 tables)
        assert bool(((a - b).abs() <= 2.0 ** -7 * a.abs().clamp(min=a.abs().mean().item())).all())
