"""The library on the system's HIP runtime: the test processes import torch first and share its runtime, so these run
programs without it, or with it second, in processes of their own."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PATHS = [ROOT, os.path.join(ROOT, "symmetrix-xl_amd")]


def _child(script):
    return subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = %r\n%s" % (PATHS, script)],
                          capture_output=True, text=True, timeout=110, cwd=ROOT)


def test_node_operators_refuse_a_second_runtime():
    """The evaluators first and torch after them: two runtimes, which symmetrix.node_ops says and does not load."""
    out = _child("import symmetrix.calculator\n"
                 "assert 'torch' not in sys.modules\n"
                 "import torch\n"
                 "try:\n"
                 "    import symmetrix.node_ops\n"
                 "except ImportError as e:\n"
                 "    print('refused:', e)\n")
    assert out.returncode == 0, out.stderr[-4000:]
    assert "refused: two HIP runtimes are loaded" in out.stdout and "import torch before symmetrix" in out.stdout


@pytest.mark.gpu
def test_evaluator_without_torch():
    """Energy, forces and stress of the tiny model against the oracle, on the system's runtime alone."""
    out = _child("import __graft_entry__\n"
                 "__graft_entry__.smoke()\n"
                 "assert 'torch' not in sys.modules\n"
                 "maps = {l.split(None, 5)[5].strip() for l in open('/proc/self/maps') if 'libamdhip64.so' in l}\n"
                 "print('runtimes', len(maps), any('torch' in m for m in maps))\n")
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    assert "smoke: energy" in out.stdout and "runtimes 1 False" in out.stdout
