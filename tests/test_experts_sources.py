"""What can be seen of the kernels around experts without running them: that each waiter is counted, so that no barrier moves on two phases while a warp waits for one."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trellis-everywhere_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def kernel(text, name):
    """The body of a kernel: from its name to the end of its braces."""
    at = text.index("{", text.index(f" {name}("))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if not depth:
            return text[at:i + 1]


def phases_missed(waiters, arrivals, uses):
    """Whether, in any order of events, a warp that waits for phase u of a buffer's `full` barrier may find phase u + 1 complete.  Of `waiters` warps, the first `arrivals` arrive on `empty` when
    they have seen their phase; phase u + 1 of `full` completes when all of these have seen phase u."""
    states, seen = [(0, (0,) * waiters)], set()                # (phases of `full` complete, phases that each waiter has seen)
    while states:
        full, of = states.pop()
        if (full, of) in seen:
            continue
        seen.add((full, of))
        if any(full - w > 1 for w in of):
            return True
        if full < uses and all(w >= full for w in of[:arrivals]):
            states.append((full + 1, of))
        states += [(full, of[:i] + (w + 1,) + of[i + 1:]) for i, w in enumerate(of) if w < full]
    return False


def test_every_warp_that_waits_for_sums_is_counted():
    """Of eight warps that cut x up, four take sums; the others wait for them before they cut the next rows up.  Only if all eight arrive can none be two phases behind, where parity answers wrongly."""
    body = kernel(source("tcq_microscale_grouped.cu"), "tcq_ms_grouped_few_kernel")
    count = re.search(r"mbar_init\(smem_u32\(&sum_empty\[s\]\), (\w+)\)", body).group(1)
    assert count in ("4", "kCutters")
    arrivals = 8 if count == "kCutters" else int(count)
    assert len(re.findall(r"mbar_arrive\(smem_u32\(&sum_empty\[buf\]\)\)", body)) == (2 if arrivals == 8 else 1)
    assert phases_missed(8, 4, 3) and not phases_missed(8, arrivals, 3)


def test_kernels_that_begin_early_have_no_read_only_loads():
    """Read-only loads are defined for memory that nobody writes while the kernel runs, and these kernels run while the one before still writes; what is loaded by assembly stays where it stands."""
    around = [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and ("experts" in f or "grouped" in f or "groups" in f or "epilogue" in f or "programmatic" in f)]
    assert len(around) >= 8 and {"tcq_experts.cu", "tcq_microscale_grouped.cu", "tcq_microscale_grouped_many.cu", "tcq_microscale_epilogue.cuh", "tcq_microscale_groups.cuh"} <= set(around)
    for f in os.listdir(CSRC):
        if f.endswith((".cu", ".cuh")) and "launch_programmatic(" in source(f):
            assert f in around
    for f in around:
        text = source(f)
        assert not re.search(r"__ldg|\.nc\b|__restrict__", text), f
        for load in re.finditer(r"asm( volatile)?\((?:\s*\"[^\"]*\")*?\s*\"[^\"]*\bld\.(?:relaxed\.gpu\.)?global[^;]*;", text):
            assert load.group(1), (f, load.group(0))


def test_workspaces_of_the_most_tokens():
    """Counts of every chunk, 148 of them at most, up to the last number of tokens that is taken."""
    from trellis_b200 import _lib
    size = _lib.lib().tcq_route_workspace_bytes
    for tokens in (148 * 32, 148 * 32 + 1, 1 << 30, (1 << 31) - 149, (1 << 31) - 148, (1 << 31) - 147, (1 << 31) - 2, (1 << 31) - 1):
        chunk = -(-tokens // 148)
        assert size(tokens, 7) == -(-tokens // chunk) * 7 * 4
