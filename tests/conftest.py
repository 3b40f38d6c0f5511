import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(__file__))

import _oracle  # noqa: E402


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) CUDA device")


# Compared with the reference's own runtime, built from its sources.
WITH_REFERENCE = {"test_greedy_ids_identical_to_reference", "test_model_reload_releases_resident_weights",
                  "test_sampled_decode_through_reference_loop_matches", "test_device_greedy_decode_matches_reference",
                  "test_device_sampled_decode_matches_reference"}


def pytest_collection_modifyitems(items):
    """Where that build is absent these fail; they come last then, so that a run that stops at the first failure
    has made the others."""
    if not (_oracle.ORACLE_DIR / "_ref" / "libedgexpu_ref_runtime.so").exists():
        items.sort(key=lambda item: getattr(item, "originalname", item.name) in WITH_REFERENCE)


@pytest.fixture(scope="session")
def port():
    return _oracle.Port()


@pytest.fixture(scope="session")
def ref():
    if not _oracle.ensure_ref():
        pytest.skip("reference oracle library not built (oracle/_ref) and reference sources absent")
    return _oracle.Ref(_oracle.REF_AVX2)


@pytest.fixture(scope="session")
def ref_scalar():
    if not _oracle.ensure_ref():
        pytest.skip("reference oracle library not built (oracle/_ref) and reference sources absent")
    return _oracle.Ref(_oracle.REF_SCALAR)


@pytest.fixture(scope="session")
def pkg():
    return _oracle.load_pkg()


@pytest.fixture(scope="session")
def gpu(pkg):
    """The CUDA C ABI bound to cuda:0 (GPU tests only)."""
    pkg.init(0)
    yield pkg
    pkg.shutdown()
