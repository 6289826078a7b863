"""What the ctypes binding of the fused operators refuses before a pointer reaches a kernel, which takes it for what the sizes say.  On host
tensors: a call that nothing else is wrong with is refused for those, last."""
import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32
M, N, H = 6, 24, 16


@pytest.fixture()
def K(built, monkeypatch):
    from orion_b200 import kernels

    class Untouched:
        def __getattr__(self, name):
            raise AssertionError("%s was reached" % name)
    monkeypatch.setattr(kernels, "lib", lambda: Untouched())
    return kernels


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


RNG = z(2, dtype=torch.int64)
GOOD = {
    "linear_act": dict(x=z(M, H), w=z(N, H), bias=z(N), residual=z(M, N), act="gelu", p=0.1, rng=RNG),
    "linear_act_backward": dict(dy=z(M, N), slope=z(M, N, dtype=torch.float16), x=z(M, H), w=z(N, H), act="gelu", p=0.1, rng=RNG),
    "dropout": dict(x=z(M, N), p=0.1, rng=RNG, residual=z(M, N)),
    "linear_cross_entropy": dict(x=z(M, H), w=z(N, H), target=z(M, dtype=torch.int64)),
    "linear_cross_entropy_backward": dict(x=z(M, H), w=z(N, H), target=z(M, dtype=torch.int64), lse=z(M, dtype=F32), grad=z(M, dtype=F32), count=z((), dtype=F32)),
}
HALF, I32 = torch.float16, torch.int32
BAD = {
    "linear_act": [("x", z(M, H + 8)), ("x", z(M, H, dtype=F32)), ("x", z(H, M).T), ("w", z(N, H, dtype=HALF)), ("x", z(2, 3, H)), ("bias", z(N - 1)),
                   ("bias", z(N, dtype=HALF)), ("bias", z(2 * N)[::2]), ("residual", z(M, N - 1)), ("residual", z(M, N, dtype=F32)), ("residual", z(N, M).T),
                   ("residual", z(1, N)), ("rng", None), ("rng", z(1, dtype=torch.int64)), ("rng", z(2, dtype=I32)), ("site", -1), ("site", 2 ** 31)],
    "linear_act_backward": [("dy", z(M - 1, N)), ("dy", z(M, N, dtype=F32)), ("dy", z(N, M).T), ("slope", z(M, N - 8, dtype=HALF)), ("slope", z(M, N)),
                            ("x", z(M, H - 8)), ("bias_dtype", HALF), ("rng", None), ("rng", z(2, dtype=I32)), ("site", 2 ** 32)],
    "dropout": [("x", z(N, M).T), ("x", z(M, N, dtype=HALF)), ("residual", z(M, N, dtype=F32)), ("residual", z(M - 1, N)), ("rng", None),
                ("rng", z(4, dtype=torch.int64)[::2]), ("site", -1)],
    "linear_cross_entropy": [("target", z(M - 1, dtype=torch.int64)), ("target", z(M, dtype=I32)), ("target", z(2 * M, dtype=torch.int64)[::2]),
                             ("w", z(N, H - 8)), ("x", z(M, H, dtype=F32))],
    "linear_cross_entropy_backward": [("grad", z(1, dtype=F32)), ("grad", z(M - 1, dtype=F32)), ("grad", z(M)), ("lse", z(M - 1, dtype=F32)), ("lse", z(M)),
                                      ("target", z(M - 1, dtype=torch.int64)), ("count", z(M, dtype=F32)), ("count", z(())), ("w", z(N, H, dtype=F32))],
}


@pytest.mark.parametrize("name", GOOD)
def test_host_tensors_are_refused_last(K, name):
    with pytest.raises(AssertionError, match="CUDA tensors of the current device"):
        getattr(K, name)(**GOOD[name])


@pytest.mark.parametrize("name,i", [(n, i) for n in BAD for i in range(len(BAD[n]))])
def test_tensors_that_are_not_what_the_sizes_say_are_refused(K, name, i):
    argument, value = BAD[name][i]
    with pytest.raises(AssertionError, match="expected|needs rng|bfloat16 or float32"):
        getattr(K, name)(**dict(GOOD[name], **{argument: value}))
