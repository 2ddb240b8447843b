"""Counter-based dropout (transformer.functional.fused_dropout, kernels/counter_dropout.hip): the mask against Philox4x32-7
written with Python integers, the values exactly (one product in fp32, one rounding)."""
import pytest
import torch

from beforeholiday_amd.transformer.functional import dropout_keep, fused_dropout

M = 0xFFFFFFFF


def philox(seed, ctr, rounds=7):
    c, k = [ctr & M, ctr >> 32, 0, 0], [seed & M, (seed >> 32) & M]
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & M, (a >> 32) ^ c[3] ^ k[1], a & M]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    return c


@pytest.mark.parametrize("seed", [0, 1, 0xDEADBEEF12345678, (1 << 62) - 1])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_keep_flags_are_philox(seed, p):
    want = [philox(seed, i // 4)[i % 4] < int((1 - p) * 2 ** 32) for i in range(203)]
    assert dropout_keep(seed, 203, p).tolist() == want


def test_philox_with_ten_rounds_gives_the_published_words():
    """Salmon et al.'s known answer for counter 0, key 0 pins the round function of the oracle above."""
    assert philox(0, 0, 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def expect(x, p, seed):
    keep = dropout_keep(seed, x.numel(), p).view(x.shape)
    y = x.detach().cpu().float() * torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32)
    return torch.where(keep, y, torch.zeros(())).to(x.dtype)


def check(x, p, seed):
    y = fused_dropout(x, p, seed=seed)
    assert y.dtype == x.dtype and torch.equal(y.cpu(), expect(x, p, seed))
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).to(x.dtype).to(x.device)
    (g,) = torch.autograd.grad(y, x, dy, create_graph=True)
    assert torch.equal(g.cpu(), expect(dy, p, seed))


@pytest.mark.parametrize("p", [0.1, 0.75])
def test_cpu(p):
    x = torch.randn(7, 3, 5, requires_grad=True)
    check(x, p, 77)
    assert torch.equal(fused_dropout(x.detach().t() if x.dim() == 2 else x.detach().transpose(0, 2), p, seed=5),
                       fused_dropout(x.detach().transpose(0, 2).contiguous(), p, seed=5))


def test_identity_rate_one_and_special_values():
    x = torch.randn(9, requires_grad=True)
    assert fused_dropout(x, 0.0) is x and fused_dropout(x, 0.4, training=False) is x
    y = fused_dropout(x, 1.0, seed=1)
    assert (y == 0).all() and (torch.autograd.grad(y.sum(), x)[0] == 0).all()
    bad = torch.full((64,), float("nan"))
    keep = dropout_keep(3, 64, 0.5)
    y = fused_dropout(bad, 0.5, seed=3)
    assert (y[~keep] == 0).all() and torch.isnan(y[keep]).all()


@pytest.mark.parametrize("p", [-0.1, 1.1, float("nan")])
def test_refusals(p):
    with pytest.raises(ValueError):
        fused_dropout(torch.randn(4), p)
    with pytest.raises(ValueError):
        fused_dropout(torch.arange(4), 0.5)


def test_gradient_against_differences_and_twice():
    x = torch.randn(11, dtype=torch.float64, requires_grad=True)
    f = lambda t: fused_dropout(t, 0.5, seed=9)  # noqa: E731
    assert torch.autograd.gradcheck(f, (x,)) and torch.autograd.gradgradcheck(f, (x,))


def test_seeds_are_drawn_from_the_dropout_stream():
    from beforeholiday_amd.transformer.tensor_parallel import random as tr

    saved = dict(tr._DROPOUT_SEED_GENS)
    try:
        x = torch.ones(1000)
        tr._seed_dropout_streams(11, 22)
        a, b = fused_dropout(x, 0.5), fused_dropout(x, 0.5)
        m = fused_dropout(x, 0.5, model_parallel=True)
        tr._seed_dropout_streams(11, 23)
        assert torch.equal(fused_dropout(x, 0.5), a) and not torch.equal(a, b)
        assert not torch.equal(fused_dropout(x, 0.5, model_parallel=True), m)
    finally:
        tr._DROPOUT_SEED_GENS.clear()
        tr._DROPOUT_SEED_GENS.update(saved)


# ---- GPU -----------------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 4, 8, 9, 255, 2048, 100003])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_gpu(n, p, dtype):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).cuda().requires_grad_()
    check(x, p, (1 << 61) + n)


@gpu
def test_gpu_layouts_and_alignment():
    x = torch.randn(33, 47, device="cuda")
    assert torch.equal(fused_dropout(x.t(), 0.3, seed=4), fused_dropout(x.t().contiguous(), 0.3, seed=4))
    flat = torch.randn(1001, device="cuda", dtype=torch.bfloat16)
    assert flat[1:].data_ptr() % 16
    assert torch.equal(fused_dropout(flat[1:], 0.3, seed=4), fused_dropout(flat[1:].clone(), 0.3, seed=4))
    for shape in ((0,), (3, 0)):
        e = torch.empty(shape, device="cuda", requires_grad=True)
        y = fused_dropout(e, 0.3, seed=4)
        assert y.shape == e.shape and torch.autograd.grad(y.sum(), e)[0].shape == e.shape
    with pytest.raises(ValueError):
        fused_dropout(x.double(), 0.3)


@gpu
def test_counters_past_32_bits_of_elements():
    """2^32 + 1024 elements: the last ones use counters just above 2^30 and offsets past 32 bits."""
    n = (1 << 32) + 1024
    x = torch.ones(n, device="cuda", dtype=torch.float16)
    y = fused_dropout(x, 0.5, seed=123)
    for at in (0, (1 << 31) - 64, (1 << 32) - 64, n - 128):
        want = [philox(123, i // 4)[i % 4] < 1 << 31 for i in range(at, at + 128)]
        assert (y[at:at + 128] != 0).tolist() == want
    del x, y


@gpu
def test_captured_step_draws_a_new_mask_each_replay():
    from beforeholiday_amd.utils import graph_rng

    x = torch.ones(4096, device="cuda", requires_grad=True)
    graph_rng.enable(seed=5)
    try:
        def step():
            graph_rng.new_step()
            y = fused_dropout(x, 0.5)
            return y, torch.autograd.grad(y, x, torch.ones_like(x))[0]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, g = step()
        seen = []
        for _ in range(3):
            at = int(graph_rng.step_seed())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, g)
            seen.append(y.clone())
            graph_rng.step_seed().fill_(at)
            eager = step()
            assert torch.equal(eager[0], seen[-1]) and int(graph_rng.step_seed()) == at + 1
        assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    finally:
        graph_rng.disable()
