"""GPU: embedding lookup and its gradient by sorted ids against a plain implementation in 64 bits.

Tolerances, with u = 2^-24: a lookup is one product in float and one rounding to the type (half a step:
finfo.eps / 2), so |err| <= (eps / 2 + 2 u) |v|.  A gradient row of k terms is summed in float in some fixed tree: at most
k additions, |err| <= k u sum|x| |scale|, then the product and the rounding.  Values below the type's normal range are
rounded to its smallest step (`tiny`)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope='module')
def emb(gpu_device):
    from bayes_vi_amd import embedding
    return embedding


def half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps


def make_ids(rng, n, rows, kind, dtype, dev):
    ids = {'even': lambda: rng.integers(0, rows, n),
           'skewed': lambda: np.minimum((rng.random(n) ** 6 * rows).astype(np.int64), rows - 1),
           'one': lambda: np.full(n, rows // 2),
           'padding': lambda: np.where(rng.random(n) < 0.4, rng.choice([-1, rows, rows + 7, -2 ** 31]), rng.integers(0, rows, n)),
           'nothing': lambda: np.full(n, -1)}[kind]()
    return torch.tensor(ids, dtype=dtype, device=dev)


def check_lookup(out, table, ids, scale):
    t, i = table.detach().double().cpu(), ids.long().cpu()
    keep = (i >= 0) & (i < t.shape[0])
    ref = torch.where(keep[..., None], t[torch.where(keep, i, 0)], 0.0) * scale
    e, tiny = half_step(table.dtype)
    err = (out.detach().double().cpu() - ref).abs()
    assert bool((err <= (e + 2 * U) * ref.abs() + tiny).all()), float(err.max())
    assert bool((out.detach().cpu()[~keep] == 0).all())


def check_grad(got, g, ids, rows, scale):
    g64, i = g.detach().double().cpu().reshape(ids.numel(), -1), ids.long().cpu().reshape(-1)
    keep = (i >= 0) & (i < rows)
    ref = torch.zeros(rows, g64.shape[1], dtype=torch.float64).index_add_(0, i[keep], g64[keep])
    mag = torch.zeros_like(ref).index_add_(0, i[keep], g64[keep].abs())
    count = torch.bincount(i[keep], minlength=rows)[:, None]
    e, tiny = half_step(g.dtype)
    err = (got.detach().double().cpu().reshape(rows, -1) - ref * scale).abs()
    bound = abs(scale) * (count * U * mag) * (1 + e) + (e + 2 * U) * (ref * scale).abs() + tiny
    assert bool((err <= bound).all()), (float(err.max()), int((err > bound).sum()))


SHAPES = [(1, 1, 1), (85, 4, 919), (3, 5, 2), (1000, 1, 777), (17, 64, 4097), (301, 129, 1000), (5, 1023, 300),
          (40000, 8, 5000), (70000, 3, 129), (2, 16, 70001), (12, 640, 9000)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_lookup_and_gradient(emb, gpu_device, shape, dtype):
    rows, width, n = shape
    rng = np.random.default_rng(rows * 7 + n)
    gen = torch.Generator(device=gpu_device); gen.manual_seed(n)
    for k, (kind, id_type) in enumerate([('even', torch.int64), ('skewed', torch.int32), ('padding', torch.int64),
                                         ('padding', torch.int32), ('one', torch.int32), ('nothing', torch.int64)]):
        ids = make_ids(rng, n, rows, kind, id_type, gpu_device)
        table = torch.randn(rows, width, generator=gen, device=gpu_device).to(dtype)
        check_lookup(emb.lookup(table, ids, scale=1.75), table, ids, 1.75)
        g = torch.randn(n, width, generator=gen, device=gpu_device).to(dtype)
        a = emb.lookup_grad(g, ids, rows, scale=0.375)
        check_grad(a, g, ids, rows, 0.375)
        plan = emb.LookupPlan(ids, rows)
        assert torch.equal(emb.lookup_grad(g, ids, rows, scale=0.375, plan=plan), a)     # and the same bits again


@pytest.mark.parametrize('rows', [1, 2, 200, 255, 256, 300, 70000, 3_000_000, 20_000_000])
@pytest.mark.parametrize('n', [0, 1, 63, 4096, 4097, 100_003])
def test_plan_is_the_stable_sort(emb, gpu_device, rows, n):
    gen = torch.Generator(device=gpu_device); gen.manual_seed(n + rows)
    for id_type in (torch.int32, torch.int64):
        ids = (torch.rand(n, generator=gen, device=gpu_device, dtype=torch.float64) * (rows + 2)).long() - 1
        plan = emb.LookupPlan(ids.to(id_type), rows)
        key = torch.where((ids >= 0) & (ids < rows), ids, rows)
        key, order = torch.sort(key, stable=True)
        w = (n + 63) // 64 * 64
        buf = plan.buffer.view(torch.int32)
        assert torch.equal(buf[:n].long(), order)
        assert torch.equal(buf[w:w + n].long(), key)
        start = torch.searchsorted(key, torch.arange(rows + 1, device=gpu_device))
        assert torch.equal(buf[2 * w:2 * w + rows + 1].long(), start)


def test_long_rows_are_split_and_joined(emb, gpu_device):
    """One row of most positions among thousands of short ones, over the sizes where whole blocks of sorted positions,
    and blocks of blocks, are summed beforehand."""
    gen = torch.Generator(device=gpu_device); gen.manual_seed(1)
    for n in (127, 128, 255, 256, 16384, 32768, 40000, 300_001):
        rows = 700
        ids = torch.randint(0, rows, (n,), generator=gen, device=gpu_device)
        ids[torch.rand(n, generator=gen, device=gpu_device) < 0.8] = 333
        for width in (1, 4, 7):
            g = torch.randn(n, width, generator=gen, device=gpu_device)
            check_grad(emb.lookup_grad(g, ids, rows, scale=1.0), g, ids, rows, 1.0)


def test_many_positions_in_two_rows(emb, gpu_device):
    n, rows = 4_300_003, 2
    gen = torch.Generator(device=gpu_device); gen.manual_seed(2)
    ids = torch.randint(0, 2, (n,), generator=gen, device=gpu_device, dtype=torch.int32)
    g = torch.randn(n, 2, generator=gen, device=gpu_device)
    check_grad(emb.lookup_grad(g, ids, rows), g, ids, rows, 1.0)


def test_layouts(emb, gpu_device):
    gen = torch.Generator(device=gpu_device); gen.manual_seed(3)
    ids = torch.randint(0, 50, (7, 11), generator=gen, device=gpu_device)
    base = torch.randn(50, 40, generator=gen, device=gpu_device)
    for table in (base[:, :16], base[:, 3:16], base[::2].repeat(2, 1)[:50], base.T[:40].T, base[:, 1:2],
                  base[:1].expand(50, 40), base.T.contiguous().T):
        check_lookup(emb.lookup(table, ids, scale=0.5), table, ids, 0.5)
    flat = base[:, 0]
    assert torch.equal(emb.lookup(flat, ids, scale=2.0), 2.0 * flat[ids])
    assert torch.equal(emb.lookup(base[:, 5].contiguous(), ids.T), base[:, 5][ids.T])
    g = torch.randn(7, 11, 40, generator=gen, device=gpu_device)
    for grad in (g, g[..., :16], g[..., 1:], g[:1].expand(7, 11, 40), torch.ones((), device=gpu_device).expand(7, 11, 40)):
        check_grad(emb.lookup_grad(grad, ids, 50, scale=0.5), grad, ids, 50, 0.5)
    got = emb.lookup_grad(g[..., 0], ids, 50)
    assert got.shape == (50,)
    check_grad(got, g[..., 0], ids, 50, 1.0)
    half = torch.randn(50, 41, generator=gen, device=gpu_device).half()
    for table in (half[:, 1:9], half[:, 2:8], half[:, :4]):
        check_lookup(emb.lookup(table, ids, scale=0.5), table, ids, 0.5)


def test_plan_with_ids_of_another_layout(emb, gpu_device):
    """The plan and the ids may both be used: ids that are not contiguous come in their own order."""
    gen = torch.Generator(device=gpu_device); gen.manual_seed(31)
    for n in (40, 4000):
        ids = torch.randint(0, 20, (n, 3), generator=gen, device=gpu_device).T
        g = torch.randn(3, n, 5, generator=gen, device=gpu_device)
        plan = emb.LookupPlan(ids, 20)
        a = emb.lookup_grad(g, ids, 20, plan=plan)
        check_grad(a, g, ids, 20, 1.0)
        assert torch.equal(a, emb.lookup_grad(g, ids.contiguous(), 20))


def test_no_positions_for_a_large_table(emb, gpu_device):
    none = torch.zeros(0, dtype=torch.int32, device=gpu_device)
    got = emb.lookup_grad(torch.zeros(0, 2, device=gpu_device), none, 5_000_000)
    assert got.shape == (5_000_000, 2) and not bool(got.any())


def test_no_ids(emb, gpu_device):
    table = torch.randn(5, 3, device=gpu_device, requires_grad=True)
    none = torch.zeros(0, dtype=torch.int64, device=gpu_device)
    out = emb.lookup(table, none)
    assert out.shape == (0, 3)
    out.sum().backward()
    assert torch.equal(table.grad, torch.zeros(5, 3, device=gpu_device))


def test_special_values(emb, gpu_device):
    inf, nan = float('inf'), float('nan')
    table = torch.tensor([[1., inf], [nan, -inf], [0., 3.]], device=gpu_device)
    ids = torch.tensor([0, -1, 1, 3, 2], device=gpu_device)
    out = emb.lookup(table, ids, scale=2.0).cpu()
    want = torch.tensor([[2., inf], [0., 0.], [nan, -inf], [0., 0.], [0., 6.]])
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(7.), want.nan_to_num(7.))
    # an infinite scale, and what padding carries, stay out of rows that nobody read
    g = torch.tensor([[1.], [nan], [2.], [inf], [-1.]], device=gpu_device)
    got = emb.lookup_grad(g, ids, 3, scale=2.0).cpu()
    assert got.reshape(-1).tolist() == [2., 4., -2.]
    got = emb.lookup_grad(g, torch.tensor([0, -1, 0, -1, 0], device=gpu_device), 3, scale=inf).cpu()
    assert got.reshape(-1).tolist() == [inf, 0., 0.]
    # sums whose parts leave the type's range but whose total does not: the running sum is in float
    big = torch.full((4, 1), 60000., device=gpu_device).half()
    big[2:] *= -1
    got = emb.lookup_grad(big, torch.zeros(4, dtype=torch.int32, device=gpu_device), 1)
    assert got.item() == 0.0


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_autograd(emb, gpu_device, dtype):
    gen = torch.Generator(device=gpu_device); gen.manual_seed(5)
    table = torch.randn(30, 12, generator=gen, device=gpu_device).to(dtype).requires_grad_()
    ids = torch.randint(-1, 31, (9, 5), generator=gen, device=gpu_device)
    w = torch.randn(9, 5, 12, generator=gen, device=gpu_device).to(dtype)
    out = emb.lookup(table, ids, scale=0.5)
    out.backward(w)
    check_grad(table.grad, w, ids, 30, 0.5)
    assert torch.equal(table.grad, emb.lookup_grad(w, ids, 30, scale=0.5))
    if dtype == torch.float32:
        # against differences: the map is linear, so any step serves; step 1 keeps the quotient's error at that of the
        # two sums of 45 * 12 products of size < 8 (each sum off by < 540 u 8 * 4.5)
        for r, c in ((0, 0), (7, 3), (29, 11)):
            with torch.no_grad():
                hi, lo = table.clone(), table.clone()
                hi[r, c] += 1.0
                lo[r, c] -= 1.0
                f = lambda t: (emb.lookup(t, ids, scale=0.5).double() * w.double()).sum()
                diff = float(f(hi) - f(lo)) / 2
            assert abs(diff - float(table.grad[r, c])) <= 540 * U * 8 * 4.5
    with pytest.raises(RuntimeError):
        table2 = table.detach().clone().requires_grad_()
        y, = torch.autograd.grad(emb.lookup(table2, ids).float().pow(2).sum(), table2, create_graph=True)
        y.float().sum().backward()


def test_shared_table_gradients_add(emb, gpu_device):
    """One table read twice and used directly as well."""
    gen = torch.Generator(device=gpu_device); gen.manual_seed(6)
    table = torch.randn(6, 4, generator=gen, device=gpu_device, requires_grad=True)
    a = torch.randint(0, 6, (20,), generator=gen, device=gpu_device)
    b = torch.randint(0, 6, (3,), generator=gen, device=gpu_device)
    (emb.lookup(table, a).sum() + 2.0 * emb.lookup(table, b, scale=3.0).sum() + table.sum()).backward()
    want = torch.bincount(a, minlength=6) + 6.0 * torch.bincount(b, minlength=6) + 1.0
    assert torch.equal(table.grad, want[:, None].expand(6, 4).float())


def test_refusals_on_the_device(emb, gpu_device):
    table = torch.zeros(4, 3, device=gpu_device)
    ids = torch.zeros(5, dtype=torch.int64, device=gpu_device)
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        emb.lookup(table.double(), ids)
    with pytest.raises(ValueError, match='ids are on cpu'):
        emb.lookup(table, ids.cpu())
    plan = emb.LookupPlan(ids, 4)
    with pytest.raises(ValueError, match='this plan is for'):
        emb.lookup(table, ids[:4], plan=plan)
    with pytest.raises(ValueError, match='this plan is for'):
        emb.lookup_grad(torch.zeros(5, 3, device=gpu_device), ids, 5, plan=plan)


def test_graph_replays_follow_the_inputs(emb, gpu_device):
    """Forward, sort and gradient recorded once and replayed on new ids and values, with eager work between."""
    gen = torch.Generator(device=gpu_device); gen.manual_seed(7)
    rows, width, n = 90, 20, 3000
    table = torch.randn(rows, width, generator=gen, device=gpu_device)
    ids = torch.randint(0, rows, (n,), generator=gen, device=gpu_device)
    g = torch.randn(n, width, generator=gen, device=gpu_device)
    emb.lookup(table, ids); emb.lookup_grad(g, ids, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = emb.lookup(table, ids, scale=1.5)
        grad = emb.lookup_grad(g, ids, rows, scale=1.5)
    second = torch.cuda.CUDAGraph()              # another graph of the same calls has scratch of its own
    with torch.cuda.graph(second):
        grad2 = emb.lookup_grad(out, ids, rows)
    for k in range(5):
        ids.copy_(torch.randint(-1, rows + 1, (n,), generator=gen, device=gpu_device))
        g.normal_(generator=gen)
        table.normal_(generator=gen)
        graph.replay()
        second.replay()
        want = emb.lookup(table, ids, scale=1.5), emb.lookup_grad(g, ids, rows, scale=1.5)
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])
        assert torch.equal(grad2, emb.lookup_grad(want[0], ids, rows))
        torch.cuda.synchronize()


def test_another_stream(emb, gpu_device):
    gen = torch.Generator(device=gpu_device); gen.manual_seed(8)
    ids = torch.randint(0, 1000, (200_000,), generator=gen, device=gpu_device)
    g = torch.randn(200_000, 8, generator=gen, device=gpu_device)
    want = emb.lookup_grad(g, ids, 1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [emb.lookup_grad(g, ids, 1000) for _ in range(4)]
    here = [emb.lookup_grad(g, ids, 1000) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got + here)


def test_offsets_beyond_32_bits(emb, gpu_device):
    """A table of more than 2^32 bytes and 2^31 elements, read and written at its far end."""
    rows, width = 4_200_001, 520
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device=gpu_device)
    far = torch.tensor([rows - 1, 0, rows - 2, 4_140_000, rows], device=gpu_device)
    table[far[:4]] = torch.arange(4 * width, device=gpu_device).reshape(4, width).bfloat16()
    out = emb.lookup(table, far)
    assert torch.equal(out[:4], torch.arange(4 * width, device=gpu_device).reshape(4, width).bfloat16())
    assert bool((out[4] == 0).all())
    grad = emb.lookup_grad(out, far, rows)
    assert torch.equal(grad, table)
    del table, grad
    n = 4_200_001                                       # and as many positions
    g = torch.ones(n, width, dtype=torch.bfloat16, device=gpu_device)
    ids = torch.zeros(n, dtype=torch.int32, device=gpu_device)
    ids[-3:] = 1
    g[-1] = 4.0
    got = emb.lookup_grad(g, ids, 2)
    assert bool((got[0] == torch.tensor(n - 3., device=gpu_device).bfloat16()).all()) and bool((got[1] == 6.0).all())


def test_forward_mode(emb, gpu_device):
    """A tangent of the table goes through the lookup as the table itself does: jvp(lookup) = lookup(tangent)."""
    import torch.autograd.forward_ad as fwd
    gen = torch.Generator(device=gpu_device); gen.manual_seed(12)
    ids = torch.randint(-1, 7, (9, 5), generator=gen, device=gpu_device)
    for shape in ((6, 4), (6,)):
        table, tangent = (torch.randn(*shape, generator=gen, device=gpu_device) for _ in range(2))
        want, dwant = emb.lookup(table, ids, scale=0.5), emb.lookup(tangent, ids, scale=0.5)
        keep = ((ids >= 0) & (ids < 6)).reshape(ids.shape + (1,) * (len(shape) - 1))
        assert torch.equal(dwant, torch.where(keep, 0.5 * tangent[ids.clamp(0, 5)], 0.0))
        for grad_mode in (True, False):
            for leaf in (True, False):
                with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
                    t = table.clone().requires_grad_(leaf)
                    out = fwd.unpack_dual(emb.lookup(fwd.make_dual(t, tangent), ids, scale=0.5))
                    assert torch.equal(out.primal, want) and out.tangent is not None and torch.equal(out.tangent, dwant)
        with fwd.dual_level():                       # an operand without a tangent has none afterwards either
            assert fwd.unpack_dual(emb.lookup(table, ids)).tangent is None


def test_forward_over_reverse(emb, gpu_device):
    """The Hessian of sum(lookup(table)^3) times a vector, forwards over the gradient: 6 scale^3 count table vector."""
    import torch.autograd.forward_ad as fwd
    gen = torch.Generator(device=gpu_device); gen.manual_seed(13)
    for n in (40, 3000):                             # with and without the sort
        ids = torch.randint(-1, 7, (n,), generator=gen, device=gpu_device)
        table = torch.randint(-3, 4, (6, 4), generator=gen, device=gpu_device).float().requires_grad_()
        v = torch.randint(-3, 4, (6, 4), generator=gen, device=gpu_device).float()
        count = torch.bincount(ids[(ids >= 0) & (ids < 6)], minlength=6)[:, None].float()
        with fwd.dual_level():
            dual = fwd.make_dual(table, v)
            g, = torch.autograd.grad((emb.lookup(dual, ids, scale=2.0) ** 3).sum(), dual)
            g = fwd.unpack_dual(g)
            # small whole numbers: exact
            assert torch.equal(g.primal, 24 * count * table.detach() ** 2)
            assert g.tangent is not None and torch.equal(g.tangent, 48 * count * table.detach() * v)


def test_the_gradient_is_differentiable_in_what_it_adds_up(emb, gpu_device):
    """lookup_grad is linear in grad_out: its derivative is the lookup, both ways."""
    import torch.autograd.forward_ad as fwd
    gen = torch.Generator(device=gpu_device); gen.manual_seed(14)
    for shape in ((50, 3), (50,)):
        ids = torch.randint(-1, 7, (50,), generator=gen, device=gpu_device)
        g = torch.randn(*shape, generator=gen, device=gpu_device, requires_grad=True)
        w = torch.randn((6,) + shape[1:], generator=gen, device=gpu_device)
        emb.lookup_grad(g, ids, 6, scale=0.5).backward(w)
        assert torch.equal(g.grad, emb.lookup(w, ids, scale=0.5))
        t = torch.randn(*shape, generator=gen, device=gpu_device)
        with fwd.dual_level():
            out = fwd.unpack_dual(emb.lookup_grad(fwd.make_dual(g.detach(), t), ids, 6, scale=0.5))
            assert torch.equal(out.tangent, emb.lookup_grad(t, ids, 6, scale=0.5))


WIDE = [(1, 1999, 2048), (1, 2000, 2048), (3, 1500, 1000), (2, 640, 2000), (1, 67, 2047), (5, 48, 1500), (9, 7, 2048), (2, 3, 2048),
        (4, 1, 2048), (700, 1040, 2000), (1, 4097, 65), (3, 1999, 2100), (1, 4100, 2300), (2, 2056, 5000), (40, 771, 2400)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shape', WIDE, ids=str)
def test_few_rows_of_many_positions(emb, gpu_device, shape, dtype):
    """Sizes that need no sort: rows that a workgroup shares and rows that a wave takes, in one call; columns in one
    workgroup and in several; widths and strides of every vector.  And sizes just above, with columns in several too."""
    rows, width, n = shape
    rng = np.random.default_rng(n + width)
    gen = torch.Generator(device=gpu_device); gen.manual_seed(n)
    for kind, id_type in (('one', torch.int64), ('even', torch.int32), ('skewed', torch.int64), ('padding', torch.int32)):
        ids = make_ids(rng, n, rows, kind, id_type, gpu_device)
        base = torch.randn(n, width + 3, generator=gen, device=gpu_device).to(dtype)
        for g in (base[:, :width], base[:, 1:1 + width], base[:, :width].contiguous()):
            a = emb.lookup_grad(g, ids, rows, scale=0.375)
            check_grad(a, g, ids, rows, 0.375)
            assert torch.equal(a, emb.lookup_grad(g, ids, rows, scale=0.375, plan=emb.LookupPlan(ids, rows)))


def test_wide_rows_of_many_positions_are_not_one_waves_work(emb, gpu_device):
    """2048 positions of 1999 columns in one row took 11 ms, index_add_ 0.08: within three times of it, by the fastest of
    several runs each.  Just above that number the sorted form's rows and blocks were one workgroup's work each."""
    import time
    for rows, width, n in ((1, 1999, 2048), (1, 2000, 2048), (3, 1501, 1000), (3, 1999, 2100)):
        gen = torch.Generator(device=gpu_device); gen.manual_seed(n)
        g = torch.randn(n, width, generator=gen, device=gpu_device)
        ids = torch.randint(0, rows, (n,), generator=gen, device=gpu_device)
        out = torch.empty(rows, width, device=gpu_device)
        best = []
        for f in (lambda: emb.lookup_grad(g, ids, rows), lambda: out.zero_().index_add_(0, ids, g)):
            runs = []
            for _ in range(6):
                torch.cuda.synchronize()
                start = time.perf_counter()
                for _ in range(10):
                    f()
                torch.cuda.synchronize()
                runs.append(time.perf_counter() - start)
            best.append(min(runs))
        assert best[0] < 3 * best[1], (rows, width, n, best)
