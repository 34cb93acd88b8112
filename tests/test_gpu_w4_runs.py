"""Products with 4-bit weights as a program makes them one after another."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("is_gated", [False, True])
@pytest.mark.parametrize("rows, n, k", [(129, 2048, 2048), (257, 1500, 4128), (300, 4096, 2720), (1024, 6000, 512)])
def test_pairs_multiply_the_weights_of_their_own_call(pkg, rows, n, k, is_gated):
    """The second CTA of a pair tells the first of every stage of weights that it has made: with weights that take turns, a word that came too early would
    multiply those of the call, or of the stage, before."""
    backend = pkg.CudaBackend(0)
    gen = torch.Generator("cuda").manual_seed(rows)
    weights = [pkg.quantize_w4(backend, torch.randn((n, k), generator=gen, device="cuda") * k ** -0.5, group=32, zeros=True) for _ in range(3)]
    x = torch.randn((rows, k), generator=gen, device="cuda").to(torch.bfloat16)

    def product(i):
        return pkg.gated_w4(backend, x, weights[i], weights[(i + 1) % 3]) if is_gated else pkg.linear_w4(backend, x, weights[i])

    first = []
    for i in range(3):
        first.append(product(i))
        torch.cuda.synchronize()
    assert not torch.equal(first[0], first[1])
    turns = [product(i % 3) for i in range(150)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, first[i % 3]) for i, t in enumerate(turns))
    assert backend.poll_wait_timeouts() == 0
