"""8-bit products whose device waits run out: results that nothing can take for good ones, a status word, and an end."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture
def unanswered():
    """Switches the waits of the launches that follow to something that never comes."""
    from rngd_pd import _lib, fp8
    yield lambda on: _lib.call("rngd_f8_unanswered", on)
    _lib.call("rngd_f8_unanswered", 0)
    torch.cuda.synchronize()
    fp8.device_status()  # reading clears it


def _operands(M, K, Ns, seed=0):
    from rngd_pd import fp8
    g = torch.Generator().manual_seed(seed)
    a = fp8.quantize(torch.randn(M, K, generator=g).cuda())
    return a, [fp8.quantize_weight((torch.randn(N, K, generator=g) * 0.02).cuda()) for N in Ns]


# few rows of each tile, K cut over clusters and not, more groups than the tensor memory holds; pairs of two and of many groups
@pytest.mark.parametrize("M,N,K,dt", [(3, 200, 4100, "bf16"), (7, 37000, 1100, "fp32"), (20, 333, 2100, "fp16"),
                                      (40, 1111, 2100, "fp32"), (100, 1111, 2100, "bf16"),
                                      (300, 515, 260, "fp32"), (600, 515, 1300, "bf16")])
def test_products_are_lost_and_say_so(unanswered, M, N, K, dt):
    from rngd_pd import fp8
    a, (b,) = _operands(M, K, (N,))
    want = fp8.matmul(*a, *b, dtype=DT[dt])
    room = torch.full((M + 1, N + 8), 7.0, dtype=DT[dt], device="cuda")
    torch.cuda.synchronize()
    fp8.device_status()
    unanswered(1)
    got = fp8.matmul(*a, *b, dtype=DT[dt], add=want, out=room[:M, :N])
    unanswered(0)
    torch.cuda.synchronize()
    assert torch.all(got.isnan())
    assert torch.all(room[M] == 7.0) and torch.all(room[:, N:] == 7.0)
    assert fp8.device_status() != 0 and fp8.device_status() == 0
    assert torch.equal(fp8.matmul(*a, *b, dtype=DT[dt]), want)  # the next call is none the worse
    torch.cuda.synchronize()
    assert fp8.device_status() == 0


@pytest.mark.parametrize("M,N,K", [(3, 200, 4100), (20, 300, 2100), (40, 333, 2100), (300, 260, 640)])
def test_gate_and_up_are_lost_and_say_so(unanswered, M, N, K):
    from rngd_pd import fp8
    a, (g, u) = _operands(M, K, (N, N))
    want = fp8.matmul_swiglu(*a, *g, *u)
    torch.cuda.synchronize()
    fp8.device_status()
    unanswered(1)
    q, s = fp8.matmul_swiglu(*a, *g, *u)
    unanswered(0)
    torch.cuda.synchronize()
    assert torch.all(q.float().isnan()) and torch.all(s.isnan())
    assert fp8.device_status() != 0
    again = fp8.matmul_swiglu(*a, *g, *u)
    assert torch.equal(again[0].float(), want[0].float()) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("M", [3, 300])
def test_the_engines_status_is_another_one(unanswered, M):
    """A lost product is none of a beam search's, and what a search reads and clears keeps nothing from the product's caller."""
    from rngd_pd import _lib, fp8
    a, (b,) = _operands(M, 1100, (300,))
    torch.cuda.synchronize()
    _lib.device_status(), fp8.device_status()
    unanswered(1)
    y = fp8.matmul(*a, *b)
    unanswered(0)
    assert _lib.device_status() == 0
    code = fp8.device_status(reset=False)
    assert code != 0 and fp8.device_status() == code and fp8.device_status() == 0
    assert torch.all(y.isnan())


def test_no_other_wait_ran_out():
    """Products of every tile, of many launches in a row: nobody gave up."""
    from rngd_pd import fp8
    for M, N, K in ((1, 4096, 4096), (30, 1000, 4096), (60, 2000, 2048), (128, 1000, 8192), (300, 1500, 4096)):
        a, (g, u) = _operands(M, K, (N, N))
        for _ in range(20):
            fp8.matmul(*a, *g)
            fp8.matmul_swiglu(*a, *g, *u)
    assert fp8.device_status() == 0
