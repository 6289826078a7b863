"""Ways out of the fused layer's epilogue, read from the sources: see test_kernel_waits_host.py."""
import os
import re

from tests.test_kernel_waits_host import KERNELS, _block, _roles


def test_an_epilogue_warp_that_gives_up_leaves_no_residual_copy_behind():
    """A warp asks for the residual of a turn before it waits for the accumulator, and for that of the next turn at the end of a turn.  Where
    it gives up, the CTA's shared memory may go: every way out of the walk over the tiles waits for the copy first."""
    roles = _roles("gemm_bf16.cu")
    epilogue = roles[roles.index("bool ahead = false;"):]
    epilogue = epilogue[:epilogue.index("bulk_wait_group<0>()")]
    ways_out = [m.start() for m in re.finditer(r"if \(!\*abort_flag\)", epilogue)]
    assert len(ways_out) == epilogue.count("abort_flag))") == 2   # the accumulator, the residual
    for at in ways_out:
        rest = epilogue[at:]
        assert "mbar_wait_landed(&ctl->res_full[warp - 2][slab_i & 1], (slab_i >> 1) & 1, clock64());" in rest[:rest.index("break;")]


def test_the_turn_given_up_on_is_the_one_whose_copy_is_under_way():
    """gm_epilogue_act counts turns in the caller's slab_i, gives up at one place, while it waits for the turn's own residual, and has not
    asked for the next one by then."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(KERNELS, "gemm_epilogue.cuh")).read())
    start = text.index("__device__ __forceinline__ bool gm_epilogue_act(")
    assert "uint32_t& turn" in text[start:text.index("{", start)]
    body = _block(text, start)
    assert body.count("return false") == 1
    gave_up = body.index("if (!mbar_wait_warp(&bars[turn & 1], (turn >> 1) & 1, abort_flag)) return false;")
    assert body.count("gm_residual_ahead") == 1 and body.index("gm_residual_ahead") > gave_up and body.count("turn++") == 1
