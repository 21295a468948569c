"""A kernel that lets its successor start before it has its tensor memory must leave no room on its SM for a block that allocates some: that one would keep columns
while it waits for the kernel in front of it, which waits for them.  Read from the sources and the plans of the products."""
import glob
import os
import re

from test_gemm_plan_host import CSRC, RESERVE, SM, driver, plans      # noqa: F401 (fixtures)


def _source(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


def test_nobody_beside_a_block_that_waits_for_columns(plans):      # noqa: F811
    allocate = {os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.cu")) if re.search(r"\btmem_alloc\(", _source(p))}
    assert allocate == {"gemm_tc.cu", "tree_attn.cu"}
    text = _source(os.path.join(CSRC, "tmem.cuh"))
    least, sm, block = (eval(re.search(r"\b%s = ([\d* ]+)" % n, text).group(1)) for n in ("TMEM_SHARED", "SM_SHARED", "BLOCK_SHARED"))
    assert (sm, block) == (SM, RESERVE)
    assert min(p[2] for p in plans) >= least
    # the products signal behind their allocation; the attention of trees before it, and asks for too much for a neighbour
    for body in re.findall(r"tmem_alloc\(sa\(&ctl\.tmem_base\), tmem_cols\);.*?\n  if \(warp == 0\)", _source(os.path.join(CSRC, "gemm_tc.cu")), re.S):
        assert "launch_dependents();" in body
    tree = _source(os.path.join(CSRC, "tree_attn.cu"))
    assert re.search(r"static_assert\(tensor_smem\(\) \+ tc::TMEM_SHARED \+ 2 \* tc::BLOCK_SHARED > tc::SM_SHARED", tree)
