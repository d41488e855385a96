"""Calls on a stream that is not torch's current one: what they allocate must not be memory that pending work of the
current stream still writes."""
import pytest

from example_matmul_metal4_b200 import sync_check
from example_matmul_metal4_b200.attention import AttentionDimensions, AttentionPlan
from example_matmul_metal4_b200.conv import WEIGHTS_HWIO, WEIGHTS_OHWI, Conv2DDimensions, ConvPlan, permute_weights
from example_matmul_metal4_b200.gemm import BuildOptions, GEMMDimensions, GemmPlan, splitk_finalize

pytestmark = pytest.mark.gpu


def _calls(dev):
    """name -> call(stream), and the sizes in bytes of what the calls allocate beside their results."""
    import torch

    def half(*shape):
        return torch.randn(shape, device=dev).half()

    attn = AttentionPlan(AttentionDimensions(300, 400, 64, 4, 2))
    Q, K, V = half(1, 4, 300, 64), half(1, 2, 400, 64), half(1, 2, 400, 64)
    lse = torch.empty(attn.lse_shape(), device=dev)
    O, dO = attn.run(Q, K, V, lse=lse), half(1, 4, 300, 64)
    gemm = GemmPlan(GEMMDimensions(256, 384, 512), bias=False)
    A, B = half(*gemm.a_shape()), half(*gemm.b_shape())
    C32 = torch.randn(256, 384, device=dev)
    conv = ConvPlan(Conv2DDimensions(1, 16, 16, 64, 64, 3, 3))
    x, w = half(*conv.in_shape), half(3, 3, 64, 64)
    torch.cuda.synchronize()
    return {
        "attention": lambda s: attn.run(Q, K, V, stream=s),
        "attention backward": lambda s: attn.backward(Q, K, V, O, dO, lse, stream=s),
        "gemm": lambda s: gemm.run(A, B, stream=s),
        "gemm partial": lambda s: gemm.partial(A, B, stream=s),
        "split-K finalize": lambda s: splitk_finalize(C32, None, stream=s),
        "conv": lambda s: conv.run(x, w, stream=s),
        "weights": lambda s: permute_weights(w, WEIGHTS_HWIO, WEIGHTS_OHWI, (64, 64, 1, 3, 3), stream=s),
    }, {"attention backward": attn.backward_workspace_bytes()}


@pytest.mark.parametrize("name", ["attention", "attention backward", "gemm", "gemm partial", "split-K finalize", "conv",
                                  "weights"])
def test_memory_freed_on_the_current_stream_with_work_pending(cuda, name):
    import torch
    calls, scratch = _calls(cuda)
    call = calls[name]
    side = torch.cuda.Stream()
    want = call(None)
    want = want if isinstance(want, tuple) else (want,)
    torch.cuda.synchronize()
    for _ in range(3):
        held = [torch.empty_like(t) for t in want for _ in range(3)]
        held += [torch.empty(scratch[name], dtype=torch.uint8, device=cuda) for _ in range(3 if name in scratch else 0)]
        torch.cuda._sleep(20_000_000)  # about 10 ms
        for t in held:
            t.fill_(77)
        del held, t
        got = call(side)
        torch.cuda.synchronize()
        for g, w in zip(got if isinstance(got, tuple) else (got,), want):
            assert torch.equal(g, w)


def test_split_k_workspace_is_zeroed_before_its_first_run_on_another_stream(cuda):
    """The zero fill of a plan's workspace must not wait behind work of the current stream that the run's stream does
    not wait for. Small integers: fp32 sums are exact in any order."""
    import torch
    A = torch.randint(-2, 3, (256, 8192), device=cuda).half()
    B = torch.randint(-2, 3, (512, 8192), device=cuda).half()
    want = (A.float() @ B.float().T).half()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        plan = GemmPlan(GEMMDimensions(256, 512, 8192), bias=False, buildOptions=BuildOptions(splitK=8))
        assert plan.workspace_bytes > 0
        held = [torch.full((plan.workspace_bytes,), 77, dtype=torch.uint8, device=cuda) for _ in range(3)]
        with torch.cuda.stream(side):
            held += [torch.full((plan.workspace_bytes,), 77, dtype=torch.uint8, device=cuda) for _ in range(3)]
        torch.cuda.synchronize()
        del held
        torch.cuda._sleep(20_000_000)  # about 10 ms
        C = plan.run(A, B, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(C, want)
    sync_check()
