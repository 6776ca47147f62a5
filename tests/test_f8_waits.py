"""The copies into LDS of the 8-bit product are written in assembly, whose hardware waits no compiler
looks after: on gfx9 a memory instruction may read a scalar register no sooner than 5 wait states after
a vector instruction (v_readfirstlane_b32, v_readlane_b32 of a spilled scalar, a comparison) wrote it.
Here the sources' own assembly is read for that distance, over every path that leads to a copy."""
import os
import re
import subprocess

import pytest

from mensurflow_amd import build

WAIT_STATES = 5

COPY = re.compile(r"buffer_load_\w+ (?:v\d+|off), (s\[\d+:\d+\]), (\S+) .*\blds\b")


def scalars(operand):
    """The scalar registers that an operand names: s5, s[4:7], vcc."""
    if re.fullmatch(r"s\d+", operand):
        return {int(operand[1:])}
    span = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    return set(range(int(span[1]), int(span[2]) + 1)) if span else {operand}


def functions(text):
    """The instructions of each function, as (labels, operands by instruction)."""
    body, labels = None, {}
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        label = re.fullmatch(r"([\w.$]+):", line)
        if label and not label[1].startswith(".L"):
            if body:
                yield body, labels
            body, labels = [], {}
        elif label and body is not None:
            labels[label[1]] = len(body)
        elif line and not line.startswith(".") and body is not None:
            body.append(line)
    if body:
        yield body, labels


def shortest_distances(body, labels):
    """Of each copy into LDS, the fewest wait states since a vector instruction wrote a scalar that
    it reads, WAIT_STATES where none did so within that many."""
    jumps = {}
    for i, line in enumerate(body):
        op, _, target = line.partition(" ")
        if op.startswith(("s_branch", "s_cbranch")):
            jumps.setdefault(labels[target.strip()], []).append(i)
    for i, line in enumerate(body):
        copy = COPY.match(line)
        if not copy:
            continue
        reads = scalars(copy[1]) | scalars(copy[2])
        shortest, paths, seen = WAIT_STATES, [(i, 0)], {}
        while paths:
            at, waited = paths.pop()
            if waited >= shortest or seen.get(at, WAIT_STATES) <= waited:
                continue
            seen[at] = waited
            before = list(jumps.get(at, []))
            if at > 0 and not body[at - 1].startswith(("s_branch", "s_endpgm", "s_setpc")):
                before.append(at - 1)
            for j in before:
                op, _, operands = body[j].partition(" ")
                if op.startswith("v_"):
                    # The first two operands: v_add_co_u32 and its like write a scalar second.
                    written = [o.strip() for o in operands.split(",")[:2]]
                    written = written if op.startswith(("v_add_co", "v_addc_co", "v_sub_co",
                                                        "v_subb_co", "v_subrev_co",
                                                        "v_div_scale", "v_mad_u64", "v_mad_i64")) \
                        else written[:1]
                    if any(scalars(o) & reads for o in written):
                        shortest = min(shortest, waited)
                        continue
                paths.append((j, waited + (int(operands, 0) + 1 if op == "s_nop" else 1)))
        yield shortest


def assembly(source, to):
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "--cuda-device-only", "-S", str(source), "-o",
                    str(to)], check=True, capture_output=True)
    return to.read_text()


# Scalars that a vector instruction has just written, as the offset and as the resource's size.
PROBE = """
#include "f8gemm_kernel.hpp"
using namespace mfr::f8gemm;
__global__ void copies(const char* from, int* size, int* out) {
    __shared__ int to[2][256];
    const uint32_t at = __builtin_amdgcn_readfirstlane(size[threadIdx.x]);
    copy_to_lds<16>(resource(from, 64), threadIdx.x, at, to[0]);
    copy_to_lds<4>(resource(from, size[threadIdx.x + 64]), threadIdx.x, 0, to[1]);
    wait_copies<0>();
    out[threadIdx.x] = to[0][threadIdx.x] + to[1][threadIdx.x];
}
"""


@pytest.fixture(autouse=True)
def compiler():
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")


def test_the_distance_is_found():
    body = ["v_readlane_b32 s4, v1, 0", "s_mov_b32 m0, s9", "s_nop 0",
            "buffer_load_dwordx4 v0, s[4:7], s8 offen lds"]
    assert list(shortest_distances(body, {})) == [2]
    assert list(shortest_distances(body[:2] + ["s_nop 3"] + body[3:], {})) == [5]
    loop = ["s_nop 4", "s_nop 4", "buffer_load_dword v0, s[4:7], 0 offen lds",
            "v_cmp_eq_u32_e64 s[6:7], v0, v1", "s_cbranch_scc1 .L", "s_endpgm"]
    assert list(shortest_distances(loop, {".L": 2})) == [1]


def test_a_copy_waits_for_the_scalars_that_it_reads(tmp_path):
    source = tmp_path / "probe.hip"
    source.write_text(PROBE)
    found = [d for f in functions(assembly(source, tmp_path / "probe.s"))
             for d in shortest_distances(*f)]
    assert len(found) == 2 and min(found) >= WAIT_STATES, found


def test_every_copy_of_the_product_waits(tmp_path):
    source = os.path.join(build.CSRC, "f8gemm.hip")
    found = [d for f in functions(assembly(source, tmp_path / "f8gemm.s"))
             for d in shortest_distances(*f)]
    assert len(found) > 100 and min(found) >= WAIT_STATES, sorted(found)[:10]
