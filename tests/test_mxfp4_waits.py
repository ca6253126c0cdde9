"""The waits that the tiles of the MXFP4 products count by hand, in the built code: no window of tokens is read before it has landed,
whatever order the compiler has put the loads in."""
import subprocess

import pytest

import _waits


def listing(*lines, start=0x1000):
    """Lines as llvm-objdump writes them; 'branch N': to line N."""
    out = [f"{start:016x} <kernel>:"]
    for i, line in enumerate(lines):
        op, _, to = line.partition(" -> ")
        out.append(f"\t{op} // {start + 4 * i:012X}: 00000000" + (f" <kernel+0x{4 * int(to):x}>" if to else ""))
    return _waits.instructions(out)


TOKENS, OTHER = ["buffer_load_dwordx4 v1, s[0:3], 0 offen lds"] * 4, ["buffer_load_dwordx4 v[0:3], v1, s[0:3], 0 offen"]


@pytest.mark.parametrize("prologue,body,early", [
    (TOKENS * 2, ["s_waitcnt vmcnt(4)", "s_barrier", *TOKENS], False),
    (TOKENS * 2, ["s_waitcnt vmcnt(6)", "s_barrier", *OTHER * 2, *TOKENS], True),     # in front of all of them, two too few
    (TOKENS * 2, ["s_waitcnt vmcnt(6)", "s_barrier", *TOKENS, *OTHER * 2], True),     # ... the first time only
    (TOKENS * 2 + OTHER * 2, ["s_waitcnt vmcnt(6)", "s_barrier", *TOKENS, *OTHER * 2], False),
    (TOKENS * 2 + OTHER * 2, ["s_waitcnt vmcnt(6)", "s_barrier", *TOKENS], True),  # in the loop only
    (TOKENS * 2, ["s_waitcnt vmcnt(4)", "s_barrier", "s_cbranch_scc1 2 -> 16", *OTHER * 6, "s_nop 0", *TOKENS], False),
    (TOKENS * 2, ["s_waitcnt vmcnt(10)", "s_barrier", *TOKENS, "s_cbranch_scc1 7 -> 21", *OTHER * 6, "s_nop 0"], True),  # on one path
])
def test_the_walk(prologue, body, early):
    code = listing(*prologue, *body, f"s_cbranch_scc0 9 -> {len(prologue)}", "s_waitcnt vmcnt(0)", "s_barrier", "s_endpgm")
    got, barriers = _waits.barriers_met_early(code)
    assert bool(got) == early and len(barriers) == 2  # that of the loop, and the last one


def test_tiles_wait_for_every_window(tmp_path):
    from test_abi_and_host import _code_objects
    from vllm_ascend_amd import _lib

    data, kernels = open(_lib.LIB_PATH, "rb").read(), 0
    for at in _code_objects(data):
        if b"gmm_mx_tiled_kernel" not in data[at:at + (1 << 22)]:
            continue
        part = tmp_path / "code"
        part.write_bytes(data[at:at + (1 << 22)])
        text = subprocess.run(["/opt/rocm/llvm/bin/llvm-objdump", "-d", "--mcpu=gfx950", str(part)], capture_output=True, text=True).stdout
        for body in text.split("\n\n"):
            lines = body.strip().split("\n")
            if "gmm_mx_tiled_kernel" not in lines[0]:
                continue
            kernels += 1
            early, barriers = _waits.barriers_met_early(_waits.instructions(lines))
            assert not early, (lines[0], [hex(b) for b in early])
            assert len(barriers) >= 3, lines[0]  # the two windows of the loop, and the last ones
    assert kernels == 6
