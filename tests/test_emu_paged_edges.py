"""The paged operators' tests of non-finite values and of sizes at the kernels' edges, on the library's sources built as host C++ (tests/emu)
under AddressSanitizer, so that they have passed on the CPU before they run on a device."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "tests" / "emu"))
import build_emulated  # noqa: E402

needs_rocm = pytest.mark.skipif(not (Path(build_emulated.CLANG).exists() and shutil.which("gcc")), reason="needs ROCm's clang++ and gcc")
SELECTION = ["tests/test_gpu_paged_nonfinite.py", "tests/test_gpu_paged_scores.py", "tests/test_gpu_paged_handles.py", "tests/test_gpu_sample_bounds.py",
             "tests/test_gpu_paged_forms.py::test_prefill_attention_of_128_rows_a_workgroup[640-640-16-new0-prior0-1.0]",
             "tests/test_gpu_paged_forms.py::test_decode_attention_over_more_pages_than_lanes[1-2-kv_len0-1-64]",
             "tests/test_gpu_paged_forms.py::test_decode_attention_over_more_pages_than_lanes[1-2-kv_len0-1-128]"]


@needs_rocm
def test_paged_edge_tests_pass_on_the_emulated_library_under_asan(tmp_path):
    so = build_emulated.build(tmp_path / "emulated")
    r = subprocess.run([sys.executable, "-u", "-m", "pytest", *SELECTION, "-m", "gpu", "-x", "-q", "-n", "4", "-p", "no:cacheprovider"],
                       cwd=ROOT, env=build_emulated.environment(so, "address"), capture_output=True, text=True, timeout=1500)
    tail = r.stdout[-4000:] + r.stderr[-4000:]
    assert "Sanitizer" not in r.stdout + r.stderr, tail
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and "failed" not in r.stdout, tail
