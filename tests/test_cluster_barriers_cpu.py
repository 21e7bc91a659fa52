"""Kernels whose CTAs reach into one another's shared memory: on every way to the first such access all CTAs of the cluster are known to have
begun, and on every way from the last one to the end of the kernel they are known to be done.  Read from the source: where the rule is
broken a run on a GPU may fault, or may pass for years."""
import os
import re

import pytest

import iian_b200.csrc as csrc

HERE = os.path.dirname(csrc.__file__)
ACCESS = re.compile(r"(?:ld|st)\.shared::cluster\.")
BARRIER = re.compile(r"\b(cluster_sync_all|cluster_wait|at_cluster_sync)\(\)")


def body(name, kernel):
    text = open(os.path.join(HERE, name)).read()
    start = text.index(kernel + "(")
    lines = text[start:].splitlines()
    for i, line in enumerate(lines):
        if line == "}":
            return [re.sub(r"//.*", "", x) for x in lines[:i]]
    raise AssertionError(f"{kernel} has no end")


def barriers(lines, pair):
    """Lines whose barrier a call passes whatever its sizes are: those that only some sizes reach do not count."""
    got = []
    for i, line in enumerate(lines):
        if not BARRIER.search(line):
            continue
        said = lines[i - 1] + line if "if" not in line and not lines[i - 1].rstrip().endswith((";", "{", "}")) else line
        if "recv_shared" in said or "p.ks == 1" in said:
            continue
        if ("if constexpr (PAIR)" in said and not pair) or ("if constexpr (!PAIR)" in said and pair):
            continue
        got.append(i)
    return got


@pytest.mark.parametrize("name,kernel,pair", [("linear_fused.cu", "linear_fused_kernel", False), ("linear_fused.cu", "linear_fused_kernel", True),
                                              ("linear_f32.cu", "linear_f32_kernel", False)])
def test_a_barrier_stands_before_the_first_access_and_behind_the_last(name, kernel, pair):
    lines = body(name, kernel)
    used = [i for i, line in enumerate(lines) if ACCESS.search(line)]
    stand = barriers(lines, pair)
    assert used and any(i < used[0] for i in stand) and any(i > used[-1] for i in stand)


def test_the_two_halves_come_in_their_order():
    """A barrier in two halves: one arrival at set-up, outside every warp's role, and one wait in front of the sends."""
    lines = body("linear_fused.cu", "linear_fused_kernel")
    arrive = [i for i, line in enumerate(lines) if "cluster_arrive()" in line]
    wait = [i for i, line in enumerate(lines) if "cluster_wait()" in line]
    roles = next(i for i, line in enumerate(lines) if "tmem_base = tmem_base_s" in line)
    joined = max(i for i, line in enumerate(lines) if "__syncthreads()" in line)
    send = next(i for i, line in enumerate(lines) if ACCESS.search(line))
    assert len(arrive) == len(wait) == 1 and arrive[0] < roles < joined < wait[0] < send


def test_no_other_source_reaches_into_a_cluster():
    """Whoever adds such a kernel adds it to the list above (attention_tc.cu: a barrier of the whole cluster directly before and after its sends)."""
    found = sorted(f for f in os.listdir(HERE) if f.endswith((".cu", ".cuh")) and ACCESS.search(open(os.path.join(HERE, f)).read()))
    assert found == ["attention_tc.cu", "linear_f32.cu", "linear_fused.cu"]
