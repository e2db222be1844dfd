"""What the tile loop's inline-asm products rely on, in the code built here.

The compiler does not see the wait states of the products (tokpath_gemm.h):
an accumulator must not be moved or written, nor a fragment come from a vector
instruction right before its product, inside the loop of the products."""

import os
import re
import subprocess

import pytest

from graspo_amd import build as B


@pytest.fixture(scope="module")
def every_kernel(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "linear.s"
    flags = [f for f in B.HIP_FLAGS if f != "-fPIC"]
    subprocess.run([B._hipcc(), *flags, "-S", "--cuda-device-only",
                    os.path.join(B.CSRC, "tokpath_linear.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    found = re.findall(r"^(_ZN3gtp3(?:lin|few)\w+):(.*?)\.Lfunc_end", out.read_text(), re.S | re.M)
    code = {}
    for name, body in found:
        lines = [x.strip() for x in body.split("\n")]
        code[name] = [x for x in lines if x and not x.startswith((";", "."))]
    return {k: v for k, v in code.items() if any("v_mfma" in x for x in v)}


@pytest.fixture(scope="module")
def kernels(every_kernel):
    # (those for few rows leave their products to the compiler)
    return {k: v for k, v in every_kernel.items() if "few_" not in k}


def registers(token):
    m = re.match(r"[va]\[(\d+):(\d+)\]$", token)
    return set(range(int(m.group(1)), int(m.group(2)) + 1)) if m else set()


def operands(line):
    return [x.strip(",") for x in line.split()[1:]]


def test_every_product_kernel_is_there(kernels):
    # four products in two types
    assert len(kernels) == 8
    for body in kernels.values():
        assert sum("v_mfma" in x for x in body) == 256  # two K steps of 128


def test_accumulators_stay_in_place(kernels):
    for name, body in kernels.items():
        at = [i for i, x in enumerate(body) if "v_mfma" in x]
        for x in body[at[0] : at[-1] + 1]:
            assert "accvgpr" not in x and "scratch" not in x, (name, x)
        for i in at:
            d, _, _, c = operands(body[i])
            assert d == c and d.startswith("a["), (name, body[i])


def test_wait_states_around_the_loop(kernels):
    for name, body in kernels.items():
        at = [i for i, x in enumerate(body) if "v_mfma" in x]
        after = body[at[-1] + 1 :]
        # nothing touches an accumulator before the three s_nop 7
        nops = [i for i, x in enumerate(after) if x == "s_nop 7"][:3]
        first = next(i for i, x in enumerate(after) if "accvgpr" in x or re.search(r"\ba\[?\d", x))
        assert len(nops) == 3 and nops[2] < first, name
        # and the zeros are written before the s_nop 7 ahead of the loop
        before = body[: at[0]]
        nop = max(i for i, x in enumerate(before) if x == "s_nop 7")
        assert not any("accvgpr" in x for x in before[nop:]), name


def test_fragments_come_from_lds(kernels):
    """No vector instruction writes a product's operand within the eight
    instructions ahead of it."""
    for name, body in kernels.items():
        for i, x in enumerate(body):
            if "v_mfma" not in x:
                continue
            _, a, b, _ = operands(x)
            wanted = registers(a) | registers(b)
            for y in body[max(0, i - 8) : i]:
                op = y.split()[0]
                if not op.startswith("v_") or "mfma" in op or op.startswith("v_cmp") or "readlane" in op:
                    continue
                to = operands(y)[0]
                wrote = registers(to) or ({int(to[1:])} if re.match(r"v\d+$", to) else set())
                assert not wrote & wanted, (name, y, x)


def test_few_rows_stores_that_a_stage_leaves(every_kernel):
    """The wait for a stage's loads lets a full stage's stores be: as many as a
    block has, times its blocks, all of them behind the loads."""
    found = {k: v for k, v in every_kernel.items() if "few_weight_kernel" in k and "Lb1" in k}
    assert len(found) == 4
    for name, body in found.items():
        stores, blocks = (4, 6) if "ELi4E" in name else (2, 3)
        at = [i for i, x in enumerate(body) if x.startswith("buffer_store_dwordx4")]
        loads = [i for i, x in enumerate(body) if x.startswith("buffer_load_dwordx4") and " lds" in x]
        # two stages, each with one loop over its blocks
        assert len(at) == 2 * stores and len(loads) == 3 * 6, (name, len(at), len(loads))
        assert loads[11] < at[0] and at[stores - 1] < loads[12] < at[stores], name
        waits = [x for x in body if x.startswith("s_waitcnt vmcnt(%d) lgkmcnt(0)" % (stores * blocks))]
        assert len(waits) == 2, name
        assert not any(x.startswith("scratch") for x in body), name
