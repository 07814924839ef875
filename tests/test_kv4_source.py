"""CPU: what can be seen from the kernels' text alone: no operator of the 4-bit cache touches memory ahead of its dependency wait."""
import glob
import os
import re

import pytest

import cabi

FILES = sorted(glob.glob(os.path.join(cabi.ROOT, "edge-fm-x_b200", "src", "operators", "kv4_*.cuh")))
WAIT, TRIGGER = "pdl_wait();", "pdl_launch_dependents();"
# what reads or writes memory that another launch may have written: helpers, pointers of the parameters, copies
MEMORY = re.compile(r"\b(entry_of|share_of|page_of|tile_of|held|many_pages|lay_out_units|pair_of|ManyWalk|raise)\s*[(<]|\b(c\.pool|c\.page_table|lens\[|bulk_copy|fetch\()"
                    r"|\bp\.(cu_rows|lens|lens_in|lens_out|q|k|v|out|starts|stats|part|part_stats|scores|images|units|many_\w+|mass_\w+|index_\w+|moves|n_moves)\s*[\[+]")


def kernels():
    out = []
    for path in FILES:
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__[^{;]*?\b(\w+_kernel)\s*\([^{]*\{", text):
            at, depth = m.end(), 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                at += 1
            out.append((m.group(1), text[m.end():at]))
    return out


def without_lambdas(body):
    """Bodies of lambdas run where they are called, not where they stand."""
    while True:
        m = re.search(r"=\s*\[&\]\s*\([^)]*\)\s*(->\s*\w+\s*)?\{", body)
        if m is None:
            return body
        at, depth = m.end(), 1
        while depth:
            depth += {"{": 1, "}": -1}.get(body[at], 0)
            at += 1
        body = body[:m.start()] + "= 0" + body[at:]


def test_every_kernel_is_looked_at():
    names = [n for n, _ in kernels()]
    assert len(names) == len(set(names)) and {"append_kernel", "read_kernel", "attend_few_kernel", "attend_merge_kernel", "attend_query_kernel", "attend_many_kernel",
                                              "attend_join_kernel", "attend_weights_kernel", "evict_select_kernel", "evict_move_kernel"} <= set(names)


@pytest.mark.parametrize("name,body", kernels(), ids=[n for n, _ in kernels()])
def test_memory_is_touched_behind_the_wait_only(name, body):
    """griddepcontrol.wait is what makes an earlier launch's writes visible to a kernel; a predecessor that has waited for itself promises its
    successor nothing.  One wait, before anything of that kind, on every path; the successor may start once it is over."""
    body = without_lambdas(body)
    assert body.count(WAIT) == 1
    ahead = body[:body.index(WAIT)]
    assert MEMORY.search(ahead) is None, MEMORY.search(ahead).group(0)
    assert "return" not in ahead and ahead.count("{") == ahead.count("}")
    assert TRIGGER not in ahead and TRIGGER in body
