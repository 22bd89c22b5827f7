"""The model operators' C entry points refuse what their kernels cannot address (no GPU needed: nothing is
launched), and what the compiler made of their kernels."""
import os
import re
import subprocess

import pytest

from dnatok_amd import _lib, build

P = 4096                                # an address that is never looked at


def scan(x_stride=8, gate_stride=8, total=64, dim=8, n_rows=1):
    L = _lib.lib()
    need = L.dnatok_gated_scan_work_bytes(total, dim)
    return L.dnatok_gated_scan(P, x_stride, P, gate_stride, 0, None, n_rows, total, dim, 0, None, P, None, None, P, need, None)


def backward(x_stride=8, gate_stride=8, dy_stride=8, total=64, dim=8):
    L = _lib.lib()
    need = L.dnatok_gated_scan_work_bytes(total, dim)
    return L.dnatok_gated_scan_backward(P, x_stride, P, gate_stride, 0, None, 1, total, dim, 0, None, P, dy_stride, None, P, P,
                                        P, None, P, need, None)


def test_negative_strides_are_refused():
    L = _lib.lib()
    calls = [scan(x_stride=-8), scan(gate_stride=-1), backward(x_stride=-8), backward(gate_stride=-8), backward(dy_stride=-8),
             L.dnatok_gated_step(P, -8, P, 8, 0, None, 2, 8, P, P, None),
             L.dnatok_gated_step(P, 8, P, -8, 0, None, 2, 8, P, P, None),
             L.dnatok_w4_matvec(P, -64, 1, P, 8, P, None, 2, 16, 64, 32, None, P, 16, 1, None),
             L.dnatok_w4_matvec(P, 64, 1, P, 8, P, None, 2, 16, 64, 32, None, P, -16, 1, None)]
    for strides in ((-40, 0, 40), (40, -40, 40), (40, 0, -40)):
        calls.append(L.dnatok_logits_process(P, strides[0], 0, 2, 40, None, None, None, None, None, None, P, strides[1], None,
                                             0, 0, None, P, strides[2], 0, None))
    assert calls == [-1] * len(calls)


def test_tokens_too_far_apart_are_refused():
    far = 2 ** 31 // 4 // 25 + 1
    assert scan(x_stride=far) < -1 and backward(dy_stride=far) < -1


@pytest.mark.parametrize("src", ["gated_scan.hip", "w4_matvec.hip", "logits.hip"])
def test_no_flat_accesses_and_no_packed_32_bit_arithmetic(src, tmp_path):
    hipcc = build.hipcc()
    if not (os.path.isabs(hipcc) and os.path.exists(hipcc)):
        pytest.skip("hipcc not found")
    out = tmp_path / (src + ".s")
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.check_call([hipcc, *flags, "-I", build.CSRC, "-S", "--cuda-device-only", "-o", str(out),
                           os.path.join(build.CSRC, src)], stderr=subprocess.DEVNULL)
    code = [line.split(";")[0].strip() for line in out.read_text().splitlines()]
    bad = [c for c in code if re.search(r"\bflat_(load|store|atomic)|\bv_pk_(add|mul|fma)_f32", c)]
    assert not bad, f"{len(bad)}, e.g. {bad[:3]}"
    # registers that a kernel keeps in scratch memory by choice: logits from and to 32 bits; bfloat16 products of 64 rows
    spilled, kernel = {}, None
    for c in code:
        if m := re.match(r"^(_Z\w+):", c):
            kernel = m.group(1)
        if re.search(r"\bscratch_store_dword", c):
            spilled[kernel] = spilled.get(kernel, 0) + 4 * {"x2": 2, "x3": 3, "x4": 4}.get(c.split()[0][-2:], 1)
    most = {"gated_scan.hip": 0, "w4_matvec.hip": 24, "logits.hip": 16}[src]
    assert max(spilled.values(), default=0) <= most, spilled
