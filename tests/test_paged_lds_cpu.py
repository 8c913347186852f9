"""The decode attention's waves write a partial result to LDS and read other lanes' values of it at once
(paged_attn.hip, `finish`).  Only a barrier of the wave says that the one comes before the other, and that
the reads are over before the next result is written there: the compiler sees each lane's addresses alone.
Here the assembly of this library's own build is walked along every branch: behind a matrix product, up to
the workgroup's next barrier, no LDS read may follow a write, and no write a read, without one of the two
barriers in between.  The results are the accesses of 16 bytes (single words are the tables of lengths, which
the workgroup's barrier before the products covers)."""
import os
import re
import subprocess

import pytest

from test_lds_reads_cpu import BRANCH, hipbuild, kernels

WAVE_BARRIER = "; wave barrier"


def blocks_of(body):
    """[(label, [instruction or WAVE_BARRIER])]"""
    out = [("", [])]
    for line in body.split("\n"):
        code = line.split(";")[0].strip()
        label = re.match(r"(\.LBB\w+):", code)
        if label:
            out.append((label.group(1), []))
        elif line.strip() == WAVE_BARRIER:
            out[-1][1].append(WAVE_BARRIER)
        elif code and not code.startswith(".") and not code.endswith(":"):
            out[-1][1].append(code)
    return out


def unordered(body):
    """LDS accesses that no barrier keeps behind those of the other kind before them, and how many
    accesses were seen behind a product."""
    blocks = blocks_of(body)
    at = {label: i for i, (label, _) in enumerate(blocks)}
    bad, seen, counted, work = set(), set(), set(), [(0, False, "")]
    while work:
        state = work.pop()
        if state in seen:
            continue
        seen.add(state)
        i, product, last = state
        for n, code in enumerate(blocks[i][1]):
            op, _, rest = code.replace("\t", " ").partition(" ")
            if code == WAVE_BARRIER:
                last = ""
            elif op == "s_barrier":
                product, last = False, ""
            elif op.startswith("v_mfma"):
                product = True
            elif product and op in ("ds_read_b128", "ds_write_b128"):
                kind = op[3:5]
                counted.add((i, n))
                if last and kind != last:
                    bad.add(f"{blocks[i][0]}: {code}")
                last = kind
            if BRANCH.fullmatch(op):
                work.append((at[rest.strip()], product, last))
            if op in ("s_branch", "s_endpgm"):
                break
        else:
            if i + 1 < len(blocks):
                work.append((i + 1, product, last))
    return bad, len(counted)


@pytest.fixture(scope="module")
def attention(tmp_path_factory):
    dst = str(tmp_path_factory.mktemp("asm") / "paged_attn.s")
    subprocess.run([hipbuild.hipcc(), *hipbuild.HIPCC_FLAGS, "--cuda-device-only", "-S",
                    os.path.join(hipbuild.CSRC, "paged_attn.hip"), "-o", dst], check=True, capture_output=True)
    return dict(kernels(open(dst).read()))


def test_a_waves_exchange_through_lds_is_ordered(attention):
    assert len(attention) == 5                         # D = 128, 256, bf16 and E4M3, the last with 4 and 8 waves
    for name, body in attention.items():
        bad, seen = unordered(body)
        assert seen > 10, name
        assert not bad, (name, sorted(bad)[:5])


def test_the_walk_finds_a_missing_barrier(attention):
    """The wave barriers taken out (in the text), one at a time."""
    for name, body in attention.items():
        parts = body.split(WAVE_BARRIER)
        assert len(parts) > 2, name
        for i in range(1, len(parts)):
            gone = WAVE_BARRIER.join(parts[:i]) + WAVE_BARRIER.join(parts[i:])
            assert unordered(gone)[0], (name, i)
