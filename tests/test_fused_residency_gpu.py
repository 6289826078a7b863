"""The CTAs an SM that the fused operators' kernels are announced with (an SM quota of q cuts a launch to q times as many) against those that
an SM holds.  A launch under a quota may then occupy no more than q SMs."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Stands in front of the CUDA runtime and of the capture library's mark: notes every launch, with what the driver says an SM holds of it.
RECORDER = r"""
#include <cuda_runtime_api.h>
#include <dlfcn.h>
#include <stdio.h>
#include <string.h>
#include <map>
#include <mutex>
#include <string>
static std::map<const void*, int> announced;
static std::string lines;
static std::mutex lock;
static int quota = 0;
template <typename F>
static F real(const char* name) {
    static void* rt = dlopen("libcudart.so.12", RTLD_LAZY | RTLD_NOLOAD);
    return (F)dlsym(rt, name);
}
static void note(const void* f, unsigned blocks, unsigned threads, size_t smem) {
    static auto occupancy = real<cudaError_t (*)(int*, const void*, int, size_t)>("cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    static auto name_of = real<cudaError_t (*)(const char**, const void*)>("cudaFuncGetName");
    std::lock_guard<std::mutex> hold(lock);
    const auto it = announced.find(f);
    const char* name = nullptr;
    if (name_of(&name, f) != cudaSuccess || !strstr(name, "ob200")) return;
    int resident = -1;
    if (occupancy(&resident, f, (int)threads, smem) != cudaSuccess) resident = -1;
    char line[2048];
    snprintf(line, sizeof line, "%s %d %d %u %d\n", name, it == announced.end() ? 0 : it->second, resident, blocks, quota);
    lines += line;
}
extern "C" int orion_capture_mark_elastic(const void* f, int ctas_per_sm) {
    std::lock_guard<std::mutex> hold(lock);
    announced[f] = ctas_per_sm;
    return 0;
}
extern "C" cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void** args) {
    static auto launch = real<cudaError_t (*)(const cudaLaunchConfig_t*, const void*, void**)>("cudaLaunchKernelExC");
    note(f, c->gridDim.x * c->gridDim.y * c->gridDim.z, c->blockDim.x, c->dynamicSmemBytes);
    return launch(c, f, args);
}
extern "C" cudaError_t cudaLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t smem, cudaStream_t st) {
    static auto launch = real<cudaError_t (*)(const void*, dim3, dim3, void**, size_t, cudaStream_t)>("cudaLaunchKernel");
    note(f, grid.x * grid.y * grid.z, block.x * block.y * block.z, smem);
    return launch(f, grid, block, args, smem, st);
}
extern "C" void recorder_quota(int q) { quota = q; }
extern "C" const char* recorder_lines() { return lines.c_str(); }
"""

RUN = r"""
import ctypes, json, sys
import torch
from orion_b200 import torch_ops
ops = torch_ops.load()
recorder = ctypes.CDLL(None)
recorder.recorder_lines.restype = ctypes.c_char_p
BF, cuda = torch.bfloat16, "cuda"
randn = lambda *s: torch.randn(*s, device=cuda).to(BF)
rng = torch.tensor([1, 2], device=cuda)

def everything():
    for M in (1, 12, 20):                                                     # few rows: straight to registers, through the ring
        for N, K in ((1024, 4096), (4096, 1024), (20000, 512)):
            ops.linear_act(randn(M, K), randn(N, K), None, None, "gelu")
        for V in (2000, 20000):
            ops.linear_cross_entropy(randn(M, 512), randn(V, 512), torch.zeros(M, dtype=torch.long, device=cuda))
    for M, N, K in ((600, 1024, 4096), (600, 1023, 4096), (2050, 520, 72), (40, 72, 64)):
        for bias in (BF, torch.float32):
            x, w, b = (t.requires_grad_(True) for t in (randn(M, K), randn(N, K), randn(N).to(bias)))
            y = ops.linear_act(x, w, b, randn(M, N), "gelu", 0.1, rng)
            torch.autograd.grad(y, (x, w, b), randn(M, N))
    for dtype in (torch.float32, BF):
        for n in (4096 * 1024, 4095):
            x = torch.randn(n + 1, device=cuda).to(dtype)
            ops.dropout(x[:n], 0.1, rng)
            ops.dropout(x[1:], 0.1, rng)
    for T, V, H in ((100, 3000, 512), (700, 5003, 136), (2000, 20000, 264)):
        x, w, target = randn(T, H).requires_grad_(True), randn(V, H).requires_grad_(True), torch.randint(0, V, (T,), device=cuda)
        target[::3] = -100
        torch.autograd.grad(ops.linear_cross_entropy(x, w, target), (x, w))

torch.autograd.set_multithreading_enabled(False)   # a quota is the calling thread's: backward passes stay in it
for q in (0, 3, 1):
    ops.set_sm_quota(q)
    recorder.recorder_quota(q)
    everything()
torch.cuda.synchronize()
print("LAUNCHES" + json.dumps(recorder.recorder_lines().decode()))
"""


def test_no_launch_takes_more_sms_than_its_quota(built, tmp_path):
    (tmp_path / "recorder.cpp").write_text(RECORDER)
    so = str(tmp_path / "recorder.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-I/usr/local/cuda/include", "-o", so, str(tmp_path / "recorder.cpp"), "-ldl"], check=True)
    run = subprocess.run([sys.executable, "-c", RUN], cwd=ROOT, env=dict(os.environ, LD_PRELOAD=so), capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-3000:]
    text = next(line for line in run.stdout.splitlines() if line.startswith("LAUNCHES"))
    launches = [line.split() for line in json.loads(text[len("LAUNCHES"):]).splitlines()]
    assert launches
    names = {l[0] for l in launches}
    for part in ("few_tiles_kernelILi1ELb0", "few_tiles_kernelILi2ELb0", "few_tiles_kernelILi4ELb0", "few_tiles_kernelILi1ELb1", "few_tiles_kernelILi2ELb1",
                 "few_tiles_kernelILi4ELb1", "few_rows_kernelILi1ELb0", "few_rows_kernelILi2ELb0", "few_rows_kernelILi4ELb0", "few_rows_kernelILi1ELb1",
                 "few_rows_kernelILi2ELb1", "few_rows_kernelILi4ELb1", "ce_rows_kernelILi4E", "ce_rows_kernelILi32E", "ce_pack", "ce_unpack", "ce_total",
                 "gemm_splitk_act", "gemm_splitk_finish4", "act_backward_kernelILb0E", "act_backward_kernelILb1E", "act_colsum_kernelIf", "act_colsum_kernelI13",
                 "dropout_kernelIfLb0E", "dropout_kernelIfLb1E", "dropout_kernelI13__nv_bfloat16Lb0E", "dropout_kernelI13__nv_bfloat16Lb1E", "gemm_bf16_kernel"):
        assert any(part in n for n in names), part
    wrong = set()
    for name, announced, resident, blocks, quota in launches:
        announced, resident, blocks, quota = int(announced), int(resident), int(blocks), int(quota)
        assert resident >= 1, name
        if announced > resident or (announced == 0 and blocks > 1) or (quota and blocks > max(1, quota * resident)):
            wrong.add((name, announced, resident, blocks if quota else None, quota))
    assert not wrong, wrong
