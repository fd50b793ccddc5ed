"""The assembly check on the scaled 8-bit matrix instruction (symmetrix-xl_amd/csrc/check_mfma_waits.py): eleven
wait states before its result is touched, and no result that overlaps an operand.  (The library's own
kernels, node_product.hip among them, are checked by test_mfma_waits.py.)"""

import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "symmetrix-xl_amd", "csrc"))
import check_mfma_waits as cw  # noqa: E402

ELEVEN = """_Zk:
\tv_mfma_scale_f32_16x16x128_f8f6f4 v[20:23], v[0:7], v[8:15], v[20:23], v16, v17 op_sel_hi:[0,0,0]
\ts_nop 10
\tv_add_f32_e32 v3, v21, v3
\ts_endpgm
"""


def _check(text):
    (name, body), = cw.split_kernels(text.split("\n"))
    return cw.findings(body, 10)


def test_scaled_mfma_asks_for_eleven_states():
    assert _check(ELEVEN) == []
    # (reported with the one that it asks more)
    assert [(reg, dist) for _, _, reg, dist in _check(ELEVEN.replace("s_nop 10", "s_nop 9"))] == [("v21", 9)]


def test_overlapping_results_are_found():
    got = _check(ELEVEN.replace("v[20:23], v[0:7], v[8:15], v[20:23]", "v[4:7], v[0:7], v[8:15], v[20:23]"))
    assert [(reg, dist) for _, _, reg, dist in got] == [("v4", 0), ("v5", 0), ("v6", 0), ("v7", 0)]
