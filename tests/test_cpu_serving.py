"""The serving operators' kernels on the CPU: the small cases of
tests/test_gpu_serving.py against the emulated library (tests/emu) under
AddressSanitizer, which reports any access outside a device allocation."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))
import build_emu_lib  # noqa: E402


@pytest.fixture(scope="module")
def emulated():
    return build_emu_lib.build()


@pytest.mark.parametrize("tests", ["refusals or nothing or read_sizes", "append or growing or partial or far or zero_and or apart",
                                   "layers or finite or flat or rotated or bad_queries or batch or very_different",
                                   "test_sdpa_paged",
                                   "verify or rejection", "serving_steps"])
@pytest.mark.parametrize("reverse", ["0", "1"])
def test_small_cases_on_the_emulator(emulated, tests, reverse):
    """SQEMU_REVERSE runs the last workgroup first."""
    if reverse == "1" and tests.startswith(("refusals", "layers")):
        pytest.skip("the order of workgroups does not enter")
    env = dict(os.environ, SQHIP_LIB=emulated, LD_PRELOAD=build_emu_lib.preload(), SQEMU_REVERSE=reverse,
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=0")
    p = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-m", "gpu", "-k",
                        f"small and ({tests})", os.path.join(HERE, "test_gpu_serving.py")], capture_output=True,
                       text=True, env=env, timeout=900)
    assert p.returncode == 0 and "AddressSanitizer" not in p.stderr, p.stdout[-4000:] + p.stderr[-4000:]
