import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (a B200); runs the sm_100a kernels")


def pytest_collection_modifyitems(items):
    """Where the reference's own sources are not built (oracle/_ref), the tests that call them fail; they run last, so that
    a run that stops at the first failure has been through all the others."""
    import oracle_bindings

    if not oracle_bindings.ref_available():
        items.sort(key=lambda item: any(name.startswith("ref_") for name in item.function.__code__.co_names)
                   if hasattr(item, "function") else False)
