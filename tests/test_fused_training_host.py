"""The fused linear layer, counter-based dropout and the loss without logits, as far as the CPU goes: the generator against the published
test vectors, refused arguments (checked before any CUDA call), workspace sizes."""
import ctypes
import os
import subprocess

import pytest
import torch

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "orion_b200", "csrc", "kernels")


@pytest.fixture(scope="module")
def K(built):
    from orion_b200 import kernels
    return kernels


@pytest.fixture(scope="module")
def ops(built):
    from orion_b200 import torch_ops
    return torch_ops.load()


SHIM = """
#include <cstdint>
#define __device__
#define __forceinline__ inline
#define __host__
static inline uint32_t __shfl_sync(uint32_t, uint32_t v, int) { return v; }
%s
extern "C" void bits(uint32_t* c, const uint32_t* k) {
    // a counter of four words as (group, step, site): the step's upper bits and the group's share word 1
    ob200::DropKey key = {k[0], k[1], c[2], c[1] & 0xFFFF0000u, c[3]};
    uint32_t out[4];
    ob200::drop_bits(key, c[0] | (unsigned long long)(c[1] & 0xFFFFu) << 32, out);
    for (int i = 0; i < 4; i++) c[i] = out[i];
}
extern "C" uint32_t mask(uint64_t seed, uint64_t step, uint32_t site, uint64_t index, uint32_t threshold) {
    const long long rng[2] = {(long long)seed, (long long)step};
    return ob200::drop_mask<32>(ob200::drop_key(rng, site), index, threshold);
}
extern "C" uint32_t rate(float p, float* scale) {
    const ob200::DropRate r = ob200::drop_rate(p);
    *scale = r.scale;
    return r.threshold;
}
"""


@pytest.fixture(scope="module")
def philox(tmp_path_factory):
    text = open(os.path.join(KERNELS, "philox.cuh")).read().replace("#include <cuda_runtime.h>", "").replace("#pragma once", "")
    d = tmp_path_factory.mktemp("philox")
    (d / "p.cpp").write_text(SHIM % text)
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-o", str(d / "p.so"), str(d / "p.cpp")], check=True)
    L = ctypes.CDLL(str(d / "p.so"))
    L.mask.argtypes = [ctypes.c_uint64, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint32]
    L.mask.restype = L.rate.restype = ctypes.c_uint32
    L.rate.argtypes = [ctypes.c_float, ctypes.POINTER(ctypes.c_float)]
    return L


def plain_bits(seed, step, site, group):
    """The four words of a group, in Python's whole numbers."""
    low = 0xFFFFFFFF
    c = [group & low, (group >> 32 & 0xFFFF) | (step >> 32 & 0xFFFF) << 16, step & low, site]
    k = [seed & low, seed >> 32 & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b & low, a >> 32 ^ c[3] ^ k[1], a & low]
        k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
    return c


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_generator_gives_the_published_words(philox, counter, key, want):
    c, k = (ctypes.c_uint32 * 4)(*counter), (ctypes.c_uint32 * 2)(*key)
    philox.bits(c, k)
    assert tuple(c) == want
    step = counter[2] | (counter[1] >> 16) << 32
    assert tuple(plain_bits(key[0] | key[1] << 32, step, counter[3], counter[0] | (counter[1] & 0xFFFF) << 32)) == want


@pytest.mark.parametrize("index", [0, 8, 16, 3, 13, 2**32 - 8, 2**35 - 3, 2**40 + 1])
def test_mask_of_consecutive_elements_crosses_groups(philox, index):
    seed, step, site, threshold = 0x123456789ABCDEF, 2**33 + 5, 7, 20000
    want = 0
    for j in range(32):
        words = plain_bits(seed, step, site, (index + j) >> 3)
        e = (index + j) & 7
        want |= int((words[e >> 1] >> (e & 1) * 16 & 0xFFFF) >= threshold) << j
    assert philox.mask(seed, step, site, index, threshold) == want


def test_probability_is_a_multiple_of_two_to_the_minus_16_and_the_factor_matches_it(philox):
    s = ctypes.c_float()
    for p in (0.0, 1e-6, 0.1, 0.25, 0.5, 0.999, 1.0 - 1e-6, 1.0):
        t = philox.rate(p, ctypes.byref(s))
        assert t == min(65536, int(ctypes.c_float(p).value * 65536 + 0.5))
        assert s.value == (ctypes.c_float(65536.0 / (65536 - t)).value if t < 65536 else 0.0)


def test_entry_points_refuse_bad_arguments_without_a_gpu(K):
    L = K.lib()
    a = 1 << 20   # an aligned address that is never touched: every call below is refused before a launch

    def act(x=a, w=a, y=a, slope=None, bias=None, act=0, p=0.0, rng=None, M=4, N=8, K=8, ldx=8, ldw=8, ld_slope=0, ws=None, nbytes=0, ctas=1):
        return L.ob200_linear_act_bf16(x, w, y, slope, bias, 0, None, act, p, rng, 0, M, N, K, ldx, ldw, ld_slope, ws, nbytes, ctas, None)
    nan = float("nan")
    for bad in (dict(act=3), dict(act=-1), dict(p=-0.1), dict(p=1.5), dict(p=nan), dict(p=0.5), dict(M=-1), dict(N=-1), dict(K=0), dict(ldx=4), dict(ldw=4),
                dict(ctas=0), dict(x=None), dict(w=None), dict(y=None), dict(act=1, slope=a, ld_slope=4), dict(act=1, slope=a, ld_slope=12), dict(slope=a, ld_slope=8)):
        assert act(**bad) == -1, bad
    for bad in (dict(x=a + 8), dict(w=a + 2), dict(y=a + 4), dict(ldx=12), dict(ldw=9), dict(act=1, slope=a + 8, ld_slope=8)):
        assert act(**bad) == -2, bad
    M, N, KK = 600, 1024, 4096
    need = L.ob200_linear_act_workspace(M, N, KK)
    assert need > 0 and need % (4 * M * N) == 0
    assert act(M=M, N=N, K=KK, ldx=KK, ldw=KK, ws=a, nbytes=need - 1) == -3
    assert act(M=M, N=N, K=KK, ldx=KK, ldw=KK, ws=None, nbytes=need) == -3
    assert act(M=0) == 0 and act(N=0) == 0

    def back(dy=a, slope=None, x=a, w=a, dx=a, dw=a, db=None, act=0, p=0.0, rng=None, M=4, N=8, K=8, ldx=8, ldw=8, ld_slope=0, ws=a, nbytes=1 << 30):
        return L.ob200_linear_act_backward_bf16(dy, slope, x, w, dx, dw, db, 0, act, p, rng, 0, M, N, K, ldx, ldw, ld_slope, ws, nbytes, 1, None)
    for bad in (dict(act=2), dict(dy=None), dict(x=None), dict(w=None), dict(p=0.5), dict(act=2, slope=a, ld_slope=7), dict(K=0)):
        assert back(**bad) == -1, bad
    for bad in (dict(dy=a + 2), dict(dx=a + 2), dict(dw=a + 8), dict(ldx=9)):
        assert back(**bad) == -2, bad
    assert back(act=2, slope=a, ld_slope=8, nbytes=0) == -3 and back(db=a, M=200, ws=None) == -3
    assert back(M=0, dw=None) == 0   # dw, a sum over nothing, would be zeroed

    def drop(x=a, y=a, n=8, p=0.1, rng=a, dtype=1, ctas=1):
        return L.ob200_dropout(x, None, y, n, p, rng, 0, dtype, ctas, None)
    for bad in (dict(x=None), dict(y=None), dict(n=-1), dict(p=nan), dict(p=1.01), dict(rng=None), dict(dtype=2), dict(ctas=0)):
        assert drop(**bad) == -1, bad
    assert drop(n=0) == 0

    def ce(x=a, w=a, t=a, loss=a, lse=a, total=a, count=a, rows=4, V=9, H=8, ldx=8, ldw=8, ws=a, nbytes=1 << 30, ctas=1):
        return L.ob200_linear_cross_entropy_forward(x, w, t, loss, lse, total, count, rows, V, H, ldx, ldw, -100, 1, ws, nbytes, ctas, None)
    for bad in (dict(x=None), dict(w=None), dict(t=None), dict(loss=None), dict(lse=None), dict(count=None), dict(rows=-1), dict(V=0), dict(H=0),
                dict(ldx=4), dict(ldw=4), dict(ctas=0)):
        assert ce(**bad) == -1, bad
    assert ce(x=a + 2) == -2 and ce(ldw=12) == -2
    need = L.ob200_linear_cross_entropy_workspace(4, 9, 8)
    assert need >= 4 * 8 + 4 * 4 and ce(nbytes=need - 1) == -3 and ce(ws=None, nbytes=need) == -3
    # the scratch of a forward pass does not grow with the rows beyond a block of them
    assert L.ob200_linear_cross_entropy_workspace(10**9, 32000, 64) == L.ob200_linear_cross_entropy_workspace(65536, 32000, 64)

    def ceb(x=a, w=a, t=a, lse=a, g=a, dx=a, dw=a, rows=4, V=9, H=8, ldx=8, ldw=8, ws=a, nbytes=1 << 30, ctas=1):
        return L.ob200_linear_cross_entropy_backward(x, w, t, lse, g, 0, None, dx, dw, rows, V, H, ldx, ldw, -100, ws, nbytes, ctas, None)
    for bad in (dict(x=None), dict(w=None), dict(t=None), dict(lse=None), dict(g=None), dict(V=0), dict(H=0), dict(ldx=4), dict(ctas=0)):
        assert ceb(**bad) == -1, bad
    assert ceb(H=4, ldx=8, ldw=8) == -2 and ceb(dx=a + 2) == -2 and ceb(ldx=9) == -2
    assert ceb(nbytes=64) == -3 and ceb(ws=None) == -3
    assert ceb(dx=None, dw=None) == 0


def test_backward_of_the_loss_takes_less_scratch_than_the_logits(K):
    L = K.lib()
    rows, V, H = 8192, 32000, 1024
    # gradients of a piece's logits (at most 192 MB), copies of x and dx in bfloat16, dx in float32 and a
    # partial matrix of it: 176 + 2 x 17 + 2 x 34 MB of the 524
    assert L.ob200_linear_cross_entropy_backward_workspace(rows, V, H, 1, 1) < 0.54 * rows * V * 2
    # eight bytes for 128 columns of a row, and a copy of x: 16.4 and 16.8 MB
    assert L.ob200_linear_cross_entropy_workspace(rows, V, H) < 0.07 * rows * V * 2


def test_operators_refuse_host_tensors_and_wrong_arguments(ops):
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16)
    rng = torch.zeros(2, dtype=torch.int64)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="CUDA"):
            ops.linear_act(x.clone().requires_grad_(grad), w)
        with pytest.raises(RuntimeError, match="CUDA"):
            ops.dropout(x.clone().requires_grad_(grad), 0.1, rng)
        with pytest.raises(RuntimeError, match="CUDA"):
            ops.linear_cross_entropy(x.clone().requires_grad_(grad), w, torch.zeros(4, dtype=torch.int64))
