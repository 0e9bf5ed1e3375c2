import os
import shutil
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu via gpurun)")


def restore_preprocessors(folder):
    """The reference names its pickled Preprocessor <tag>_preproc.pyc, and what copies a tree without Python's caches leaves every *.pyc
    behind.  The four checkpoints hold the same one: preproc.pickle is that file under a name that travels."""
    for name in ("ctc", "ctc_bi", "seq2seq", "transducer"):
        target = os.path.join(folder, name + "_preproc.pyc")
        if not os.path.exists(target):
            part = "%s.%d" % (target, os.getpid())
            shutil.copyfile(os.path.join(folder, "preproc.pickle"), part)
            os.replace(part, target)


@pytest.fixture(scope="session")
def golden_dir():
    restore_preprocessors(os.path.join(GOLDEN, "ref_ckpt"))
    return GOLDEN


@pytest.fixture(autouse=True, scope="session")
def _library_options_follow_the_environment():
    """The C library reads no environment variables (include/speech_amd.h: sa_set_option); speech_amd._lib applies SA_<NAME>
    variables once, at load.  Tests switch kernel paths with monkeypatch.setenv BETWEEN calls, so here the host re-applies the
    environment whenever it changed since the last library access."""
    from speech_amd import _lib
    _lib.ENV_SYNC = True
    yield
    _lib.ENV_SYNC = False
