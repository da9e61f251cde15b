"""Rules of the serving kernels that no run can show safely, read from their
source: what happens to the others when one wait runs out, and what orders the
two ways in which memory is reached."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xpose_b200", "csrc")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"/\*.*?\*/|//[^\n]*", "", text, flags=re.S)


def body(text, name):
    """The braces' content of the function that is defined as `name`."""
    at = text.index("{", re.search(r"\b" + name + r"\((?=[^;]*?\{)", text).start())
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if not depth:
            return text[at:i + 1]
    raise AssertionError(name)


def test_tile_kernel_warps_that_part_meet_again_only_at_the_end():
    """After a wait ran out the warps leave their loops at different places: a
    barrier that counts threads among them would wait for ever."""
    kernel = body(source("serving_tile.cuh"), "attn_tile_kernel")
    parted = kernel[kernel.index("if (warp < NQ * 4)"):]
    assert not re.search(r"\bbar(rier)?\.(cta\.)?(sync|red|arrive)", parted)
    assert len(re.findall(r"__syncthreads\w*\(", parted)) == 1
    assert parted.index("__syncthreads(") > max(m.start() for m in re.finditer(r"\bat_wait\w*\(", parted))


def test_tile_kernel_row_numbers_are_none_until_given():
    """... and what a loader then reads as a row's number is a row of the cache or none."""
    kernel = body(source("serving_tile.cuh"), "attn_tile_kernel")
    assert re.search(r"G::row_off \+ i \* 4\) = AT_NONE;", kernel[:kernel.index("if (warp < NQ * 4)")])


def test_few_row_kernel_orders_its_parts_before_the_copies_that_read_them():
    """Parts are written to global memory by ordinary stores and read by bulk
    copies: a fence between the two proxies after the stores, and after the
    ticket that says they are all there, of all memory and not of shared alone."""
    kernel = body(source("serving_few.cuh"), "attn_few_kernel")
    ticket, copy = kernel.index("atomicAdd(w.tickets"), kernel.index("bulk_g2s(")
    last_part = max(m.start() for m in re.finditer(r"__stcg\(", kernel))
    assert last_part < ticket < copy
    assert "fence_proxy_async_all();" in kernel[last_part:ticket]
    assert "fence_proxy_async_all();" in kernel[kernel.index("if (s_last)", ticket + 100):copy]


def test_tile_kernel_orders_its_plan_before_the_copies_that_take_its_place():
    """The plan is made by ordinary stores in the memory where Q then arrives by
    TMA: every thread's stores, a fence, a barrier, and only then the copies."""
    kernel = body(source("serving_tile.cuh"), "attn_tile_kernel")
    assert re.search(r"at_make_plan<.*?;\s*fence_proxy_async\(\);\s*(at_fence_before\(\);)?\s*__syncthreads\(\);", kernel)
    assert kernel.index("__syncthreads();", kernel.index("at_make_plan<")) < kernel.index("at_tma(")


def test_loads_stay_behind_the_wait_for_the_kernel_before():
    """A grid that starts under the kernel before it reads nothing of that
    kernel's until it has waited: its loads in assembly are volatile, as the wait
    is, and no intrinsic stands in for them whose order the compiler may choose."""
    for name in ("serving.cuh", "serving_attn.cuh", "serving_few.cuh", "serving_tile.cuh"):
        text = source(name)
        for m in re.finditer(r"\basm\s*(volatile)?\s*\(\s*\"([^\"]*)", text):
            assert m[1] or not re.match(r"\s*(ld|cp|atom|red)\b", m[2]), m[0]
        assert not re.search(r"\b__ld(g|cg|ca|cs|lu|cv)\b", text), name


def test_tile_kernel_leaves_no_older_list_for_the_join():
    """Every way out of the kernel waits for the kernel before it, so that the
    next one may rely on that, and replaces the parts that an earlier call listed."""
    kernel = body(source("serving_tile.cuh"), "attn_tile_kernel")
    for m in re.finditer(r"\breturn;", kernel[:kernel.index("at_make_plan<")]):
        block = kernel[kernel.rindex("if (smb", 0, m.start()):m.start()]
        assert block.index("pdl_wait();") < block.index("w.heads[")
    parted = kernel[kernel.index("if (warp < NQ * 4)"):]
    assert parted.index("w.heads[") < parted.index("take()")
