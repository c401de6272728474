"""CPU: what the paged 4-bit KV cache's kernels rely on that no result shows, and its decoder's books when a step fails."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "moty_b200", "csrc")


def test_roles_take_their_registers_in_their_own_branch():
    """A warpgroup's register count is set as the first statement of a branch that whole warpgroups take: only there is the
    code that follows bounded by it.  The shares add up to what the block is launched with."""
    src = open(os.path.join(CSRC, "kv4_prompt_tc.cu")).read()
    assert len(re.findall(r"setmaxnreg\.(?:inc|dec)", src)) == 2                   # in role_registers alone
    calls = re.findall(r"(if \(warp >= \d+\)|else) \{\n\s*role_registers<(true|false), (\w+)>\(\);", src)
    assert len(calls) == len(re.findall(r"role_registers<(?:true|false)", src)) == 3
    value = lambda name: int(re.search(rf"{name} = (\d+)", src).group(1))
    edge, total = value("PT_T") // 32, 0
    for cond, more, regs in calls:
        low = int(re.search(r"\d+", cond).group()) if cond != "else" else 0
        assert low % 4 == 0 and (more == "true") == (value(regs) > value("PT_REGS"))
        total += (edge - low) * 32 * value(regs); edge = low
    assert edge == 0 and total <= value("PT_T") * value("PT_REGS") <= 65536
