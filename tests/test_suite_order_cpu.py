"""CPU: the order in which the GPU suite runs (tests/conftest.py)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_children_that_launch_cooperatively_run_first():
    """The knob tests' child processes come before every test that makes a cooperative launch in this process."""
    out = subprocess.run([sys.executable, '-m', 'pytest', '--collect-only', '-q', '-m', 'gpu', '-p', 'no:cacheprovider',
                          os.path.join('tests', 'test_gpu_kernels.py'), os.path.join('tests', 'test_gpu_knobs.py')],
                         cwd=ROOT, capture_output=True, text=True, timeout=300)
    names = [ln for ln in out.stdout.split('\n') if '::' in ln]
    knobs = [i for i, n in enumerate(names) if 'test_gpu_knobs.py::' in n]
    assert knobs and knobs == list(range(len(knobs))), out.stdout[-2000:] + out.stderr[-2000:]
    kernels = [n.split('::')[1] for n in names if 'test_gpu_kernels.py::' in n]
    assert any(n.startswith('test_gru_persistent_kernel') and 'cg' in n for n in kernels)      # (the others keep their order)
