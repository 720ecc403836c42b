"""Shared test setup: the `gpu` marker, import paths for the package and the CPU oracle."""
import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


# Tests that run the host framework (package `mira`): where it is not installed they are skipped, and say so,
# as the GPU tests that need it do; two of the files import it as they are collected.
NEEDS_MIRA = {"test_decode_cpu.py": None, "test_plan_cpu.py": None, "test_cli.py": None,
              "test_shard_gloo.py": ("test_sharded_batch_matches_single_process", "test_dead_rank_fails_the_gather_instead_of_hanging")}
NO_MIRA = "MIRA host framework (package `mira`) not importable"


def _mira_missing() -> bool:
    from mira_b200.hostfw import import_mira
    try:
        import_mira()
    except ImportError:
        return True
    return False


@pytest.hookimpl(wrapper=True)
def pytest_make_collect_report(collector):
    report = yield
    if report.failed and collector.path.name in NEEDS_MIRA and _mira_missing():
        report.outcome, report.longrepr = "skipped", (str(collector.path), None, NO_MIRA)
    return report


def pytest_collection_modifyitems(items):
    if not _mira_missing():
        return
    for item in items:
        names = NEEDS_MIRA.get(item.path.name, ())
        if names is None or item.name in names:
            item.add_marker(pytest.mark.skip(reason=NO_MIRA))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an sm_100 GPU and the built libmira_cuda.so")


@pytest.fixture(scope="session")
def cuda_device():
    """Selects device 0 through the C ABI; fails (does not skip) when no GPU is usable, so a GPU
    run can never pass on a silent fallback."""
    from mira_b200 import _lib
    from mira_b200.device import set_device
    assert _lib.device_count() > 0, "no CUDA device visible to libmira_cuda.so"
    set_device(0)
    return 0
