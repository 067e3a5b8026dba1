import os
import shutil
import sys
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")
    # The programs that tests start (some hundreds, each imports torch) share compiled modules for the run. Where the
    # environment keeps Python from writing any, each compiled a thousand files anew: 1.3 of its 2 seconds of importing.
    config.compiled_modules = tempfile.mkdtemp(prefix="tgo_tests_pyc_")
    os.environ["PYTHONPYCACHEPREFIX"] = config.compiled_modules
    os.environ.pop("PYTHONDONTWRITEBYTECODE", None)


def pytest_unconfigure(config):
    shutil.rmtree(getattr(config, "compiled_modules", ""), ignore_errors=True)


def pytest_collection_modifyitems(config, items):
    import torch
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
