"""The cache in pages and the sampling on the library's sources built as host C++ (tests/emu): bad page ids, lengths beyond the table,
stale NaN behind a sequence's end and the refusals run here first, under AddressSanitizer, and the kernels that pass data
between waves under the race detector."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "tests" / "emu"))
import build_emulated  # noqa: E402

needs_rocm = pytest.mark.skipif(not (Path(build_emulated.CLANG).exists() and shutil.which("gcc")), reason="needs ROCm's clang++ and gcc")
SAMPLING = ["tests/test_gpu_sample.py::test_sampling[1.3-0-0.9-0.05-1000-5-None]", "tests/test_gpu_sample.py::test_sampling[2.0-7-0.3-0.5-1025-3-2000]",
            "tests/test_gpu_sample.py::test_sampling[0.7-40-0.95-0.0-32000-3-None]", "tests/test_gpu_sample.py::test_infinities_and_nans[0]", "tests/test_gpu_sample.py::test_infinities_and_nans[33000]",
            "tests/test_gpu_sample.py::test_thousands_of_equal_or_coarse_logits[0]", "tests/test_gpu_sample.py::test_edges_of_the_random_number_and_of_the_settings", "tests/test_gpu_sample.py::test_sampling[0.7-40-0.95-0.0-70001-2-70004]", "tests/test_gpu_sample.py::test_sampling[1.3-0-0.9-0.05-70001-2-70004]",
            "tests/test_gpu_sample.py::test_sampling_refuses_what_it_cannot_do"]
PAGED_RACES = ["tests/test_gpu_paged.py::test_append_in_place_equals_append_beside", "tests/test_gpu_paged.py::test_decode_attention[3-6-16-kv_len9-128]",
               "tests/test_gpu_paged.py::test_decode_attention[1-17-16-kv_len7-64]", "tests/test_gpu_paged.py::test_prefill_attention[1-2-16-new8-prior8-128]",
               "tests/test_gpu_paged.py::test_prefill_attention[1-12-16-new6-prior6-64]"]


def run(so, kind, selection, workers):
    args = ["-n", str(workers)] if workers else ["-s"]
    r = subprocess.run([sys.executable, "-u", "-m", "pytest", *selection, "-m", "gpu", "-x", "-q", *args, "-p", "no:cacheprovider"],
                       cwd=ROOT, env=build_emulated.environment(so, kind), capture_output=True, text=True, timeout=1500)
    tail = r.stdout[-4000:] + r.stderr[-4000:]
    assert "Sanitizer" not in r.stdout + r.stderr, tail
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and "failed" not in r.stdout, tail


@needs_rocm
def test_paged_and_sampling_tests_pass_on_the_emulated_library_under_asan(tmp_path):
    run(build_emulated.build(tmp_path / "emulated"), "address", ["tests/test_gpu_paged.py", *SAMPLING], 4)


@needs_rocm
def test_paged_and_sampling_tests_show_no_race_between_waves(tmp_path):
    run(build_emulated.build(tmp_path / "emulated", sanitizer="thread"), "thread", [*PAGED_RACES, SAMPLING[0], SAMPLING[1], SAMPLING[-2]], 0)
