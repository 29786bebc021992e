"""CPU: `from nedo_gpu import *` brings the descriptors that a caller fills for the paged cache and for drafts."""
import nedo_gpu


def test_descriptors_are_exported():
    assert {"KvCache", "KvBatch", "Drafts"} <= set(nedo_gpu.__all__)
    assert all(hasattr(nedo_gpu, n) for n in nedo_gpu.__all__)
