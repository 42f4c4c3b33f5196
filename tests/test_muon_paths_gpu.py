"""Newton-Schulz and Muon on every way through the kernels: one block per matrix, A A and B Y in one
launch, short and long sums, small and large tiles, steps that share a product; views, graphs and
streams on each; matrices whose offsets pass 32 bits."""
import pytest
import torch

from support.muon_oracle import NS, exact, gradient, rel, tolerance
from test_muon_gpu import DEV, _muon_oracle, _Net, _wide

pytestmark = pytest.mark.gpu

# [batch,] m, n: one block per matrix up to its last row and column; one launch for A A and B Y, in
# one round of blocks and in more; then matrices of more rows
SMALL = [(1, 16, 16), (1, 17, 33), (3, 33, 48), (2, 48, 49), (1, 10, 900), (1, 32, 1088), (1, 64, 448), (1, 96, 160),
         (2, 128, 128), (1, 128, 160), (1, 5, 4096), (40, 12, 20)]
MIDDLE = [(1, 128, 161), (1, 20, 1200), (1, 1, 5000), (3, 100, 700), (2, 65, 2000), (1, 128, 4100), (1, 100, 17000),
          (20, 70, 1000)]
LARGE = [(1, 129, 129), (1, 192, 5000), (6, 200, 300), (1, 500, 1500), (1, 520, 520), (2, 700, 1000), (1, 1000, 4000),
         (12, 512, 512), (1, 1100, 2100)]
KINDS = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["fp32", "bf16", "fp16"]


def _close(x, y, precision=None):
    for a, b in zip(x.reshape(-1, *x.shape[-2:]), y.reshape(-1, *y.shape[-2:])):
        assert rel(b, exact(a, device=DEV)) <= tolerance(a, _wide(x.dtype, *a.shape, precision), x.dtype, device=DEV)


@pytest.mark.parametrize("dtype", KINDS, ids=NAMES)
@pytest.mark.parametrize("batch,m,n", SMALL + MIDDLE + LARGE)
def test_sizes(batch, m, n, dtype):
    from distributed_machine_learning_amd.optim import orthogonalize
    x = gradient(m, n, m + n, (batch,)).to(dtype).to(DEV)[:3]
    _close(x, orthogonalize(x))
    x = x.transpose(1, 2).contiguous()
    _close(x, orthogonalize(x))


@pytest.mark.parametrize("steps,coefficients", [(1, NS), (2, NS), (3, NS), (4, NS), (6, NS), (8, NS),
                                                (4, (1.5, -0.5, 0.0)), (5, (1.875, -1.25, 0.375)),
                                                (3, [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)])])
@pytest.mark.parametrize("m,n", [(30, 50), (60, 3000), (200, 6000), (260, 300)])
def test_steps_and_coefficients(m, n, steps, coefficients):
    """Steps by themselves and steps that share a product, in runs of every length."""
    from distributed_machine_learning_amd.optim import orthogonalize
    x = gradient(m, n, 6).to(DEV)
    kw = dict(steps=steps, coefficients=coefficients)
    want = exact(x, device=DEV, **kw)
    for dtype in KINDS if coefficients is NS else KINDS[:1]:
        y = orthogonalize(x.to(dtype), **kw)
        if dtype != torch.float32:
            want = exact(x.to(dtype), device=DEV, **kw)
        assert rel(y, want) <= tolerance(x.to(dtype), _wide(dtype, m, n), dtype, device=DEV, **kw)


@pytest.mark.parametrize("tall", [False, True])
def test_the_largest_tiles(tall):
    """Products of the first terms alone over a chip full of 256 x 256 tiles, sizes that end inside one."""
    from distributed_machine_learning_amd.optim import orthogonalize
    x = torch.randn(3900, 4000, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    x = x.T.contiguous() if tall else x
    _close(x, orthogonalize(x))


@pytest.mark.parametrize("m,n", [(40, 64), (64, 40), (100, 2000), (2000, 100), (300, 520)])
@pytest.mark.parametrize("dtype", KINDS, ids=NAMES)
def test_views(m, n, dtype):
    """Every alignment of rows and starts, in memory order and transposed, and batches of them."""
    from distributed_machine_learning_amd.optim import orthogonalize
    base = gradient(m + 9, n + 13, 3, (2,)).to(dtype).to(DEV)
    before = base.clone()
    for x in (base[:, 1:m + 1, :n], base[:, :m, 1:n + 1], base[:, 2:m + 2, 4:n + 4], base[1:, :m, 2:n + 2],
              base[:, 3:m + 3, 3:n + 3].transpose(1, 2), base.flatten()[3:3 + m * n].view(m, n),
              base.flatten()[8:8 + m * n].view(n, m).T, base[0, :m, :n].expand(3, m, n)):
        _close(x, orthogonalize(x))
    assert torch.equal(base, before)
    z = torch.complex(base[0].float(), base[0].float()).conj().imag      # a view that negates
    assert z.is_neg() and torch.equal(orthogonalize(z), orthogonalize(z.clone().resolve_neg().contiguous()))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("m,n", [(12, 40), (40, 12), (128, 130), (30, 2000), (100, 3000), (3000, 100)])
def test_a_bad_matrix_leaves_its_neighbours_alone(m, n, bad):
    from distributed_machine_learning_amd.optim import orthogonalize
    x = gradient(m, n, 4, (3,)).to(DEV)
    good = orthogonalize(x)
    x[1, m // 2, n // 3] = bad
    x[2] = 0
    y = orthogonalize(x)
    assert torch.equal(y[0], good[0]) and torch.equal(y[2], x[2]) and bool(torch.isnan(y[1]).all())


@pytest.mark.parametrize("batch,m,n", [(2, 64, 27), (1, 10, 512), (1, 100, 3000), (1, 500, 1500), (1, 1000, 777)])
def test_graphs_and_streams(batch, m, n):
    """Replays of two graphs between eager calls, and calls on two streams at once: the same bits."""
    from distributed_machine_learning_amd.optim import orthogonalize
    fresh = [gradient(m, n, 20 + i, (batch,)).to(DEV) for i in range(4)]
    want = [orthogonalize(v) for v in fresh]
    x = fresh[0].clone()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(orthogonalize(x))
    for v, w in zip(fresh, want):
        x.copy_(v)
        for g in graphs:
            g.replay()
        again = orthogonalize(v)
        torch.cuda.synchronize()
        assert torch.equal(again, w) and torch.equal(outs[0], w) and torch.equal(outs[1], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [orthogonalize(v) for v in fresh]
    got += [orthogonalize(v) for v in fresh]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want + want))


@pytest.mark.parametrize("shape", [(130, 200), (24, 1500), (30, 40)],
                         ids=["grouped", "one_launch_less", "one_block_each"])
def test_muon_of_many_matrices(shape):
    """More matrices than one launch takes, in an eager step and in a graph of one."""
    from distributed_machine_learning_amd.optim import Muon
    rows, cols = shape
    shapes = [s for i in range(50) for s in ((rows + i % 7, cols + 3 * (i % 11)), (3 + i,))]
    opt = Muon(_Net(shapes).to(DEV), lr=0.1, weight_decay=0.01)
    for s in opt.flat.slots:
        v = gradient(s.shape[0], s.numel // s.shape[0], s.offset % 89) if len(s.shape) > 1 else torch.ones(s.shape)
        opt.flat.grads[s.offset:s.end] = v.reshape(-1).to(DEV)
    assert len(opt.matrices) == 50

    def step_of_64_bits(run):
        p64, m64, g64 = (t.cpu().double() for t in (opt.flat.params, opt.buf, opt.flat.grads))
        run()
        torch.cuda.synchronize()
        p64, m64 = _muon_oracle(opt, p64, g64, m64, 1.0)
        assert rel(opt.flat.params, p64) <= 2e-6 and rel(opt.buf, m64) <= 4 * 2.0 ** -24

    step_of_64_bits(opt.step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        step_of_64_bits(graph.replay)
    step_of_64_bits(opt.step)


def test_muon_refuses_overlapping_buffers():
    from distributed_machine_learning_amd.ops import native
    plan = native.MuonPlan([(0, 8, 16, 1.0)], [])
    both = torch.zeros(512, device=DEV)
    p, other = torch.zeros(256, device=DEV), torch.zeros(256, device=DEV)
    for args in ((p, p, other), (p, other, p), (p, other, other), (both[:256], both[128:384], p)):
        with pytest.raises(ValueError, match="overlap"):
            native.muon_step_(plan, *args, 0.1, 0.9, 0.0)
    native.muon_step_(plan, both[:256], both[256:], p, 0.1, 0.9, 0.0)


def test_offsets_past_32_bits():
    """[130, 2^24] in fp16: 2.2e9 elements.  Y = P(A) X exactly, so slices of Y are compared with P of
    64 bits times the slices of X, the last columns among them."""
    from distributed_machine_learning_amd.optim import orthogonalize
    m, n, step = 130, 1 << 24, 1 << 20
    x = torch.empty(m, n, dtype=torch.float16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    mix = torch.randn(m, m, generator=g, device=DEV) / m ** 0.5 + torch.eye(m, device=DEV)
    for at in range(0, n, step):
        x[:, at:at + step] = (mix @ torch.randn(m, step, generator=g, device=DEV)).half()
    y = orthogonalize(x)
    a = torch.zeros(m, m, dtype=torch.float64, device=DEV)
    for at in range(0, n, step):
        part = x[:, at:at + step].double()
        a += part @ part.T
    a /= (a.diagonal().sum().sqrt() + 1e-7) ** 2
    norm = sum(float(x[:, at:at + step].double().square().sum()) for at in range(0, n, step)) ** 0.5 + 1e-7
    p, one = torch.eye(m, dtype=torch.float64, device=DEV), torch.eye(m, dtype=torch.float64, device=DEV)
    for _ in range(5):
        q = 3.4445 * one - 4.7750 * a + 2.0315 * (a @ a)
        p, a = q @ p, q @ a @ q
    # entries are about 2^-12, where fp16 has steps of 2^-22 or less: half a step is 2^-11 of the value;
    # products of 22 bits and sums in fp32 add less than that again
    for at in (0, step * 7 + 5, (1 << 31) // m - 1000, n - 5000):
        want = p @ (x[:, at:at + 5000].double() / norm)
        assert rel(y[:, at:at + 5000], want) <= 2 * 2.0 ** -11
