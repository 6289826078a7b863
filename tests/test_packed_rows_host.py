"""How the reduction of a gradient product over packed rows is cut for the rows that count (gemm_bf16.cu, gm_cut), compiled for the host:
parts that cover it, partial matrices that stay inside the scratch of the plan for all rows."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    with open(os.path.join(ROOT, "orion_b200", "csrc", "kernels", "gemm_bf16.cu")) as f:
        text = f.read()
    structs = "".join(re.search(r"struct %s \{[^}]*\};" % name, text).group(0) + "\n" for name in ("GemmCutPlan", "GemmCut"))
    start = text.index("__host__ __device__ inline GemmCut gm_cut")
    func = text[start:text.index("\n}\n", start) + 3].replace("__host__ __device__ ", "")
    d = tmp_path_factory.mktemp("cut")
    (d / "cut.cpp").write_text("constexpr int GM_BK = 64;\n" + structs + func + '''
extern "C" void cut(const int* plan, int live, int* out) {
    const GemmCutPlan c = {plan[0], plan[1], plan[2], plan[3], plan[4], plan[5], plan[6], plan[7]};
    const GemmCut r = gm_cut(c, live);
    out[0] = r.splits; out[1] = r.per_split; out[2] = r.rows;
}
''')
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-o", str(d / "cut.so"), str(d / "cut.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "cut.so")).cut

    def run(plan, live):
        out = (ctypes.c_int * 3)()
        fn((ctypes.c_int * 8)(*plan), live, out)
        return tuple(out)
    return run


@pytest.mark.parametrize("M", [257, 300, 511, 512, 700, 1143, 5000, 8192, 65536, 10**6, 2**31 - 1])
@pytest.mark.parametrize("splits,kblocks", [(1, 1), (1, 3), (1, 168), (1, 477), (3, 16), (9, 477), (16, 64), (7, 33554431)])
def test_parts_cover_the_reduction_and_fit_the_scratch(cut, M, splits, kblocks):
    per = -(-kblocks // splits)
    splits = -(-kblocks // per)
    for tiles_n in (1, 3, 16):
        for pairs in (1, 10, 74):
            plan = (M, tiles_n, kblocks, splits, per, 120 * tiles_n, (M + 63) // 64, pairs)
            for live in sorted({1, 2, 64, 255, 256, 257, M // 7 + 1, M // 2, M - 257, M - 256, M - 1, M}):
                if not 1 <= live <= M:
                    continue
                parts, deep, rows = cut(plan, live)
                assert parts >= 1 and (parts - 1) * deep < kblocks <= parts * deep      # every part has a block, together they have all
                assert live <= rows <= M
                assert parts * rows <= splits * M or parts == 1                          # partial matrices inside the plan's
                if rows < M:
                    assert rows % 256 == 0 and rows - live < 256
                else:
                    assert (parts, deep) == (splits, per) or rows % 256 == 0
