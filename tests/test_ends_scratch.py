"""Generated code: the kernels of embedding and the loss keep to their registers."""

from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_store_hazard import KERNEL_SCRATCH, _assembly

SOURCES = ("embedding.hip", "cross_entropy.hip")


@pytest.fixture(scope="module")
def scratch(tmp_path_factory):
    """Scratch bytes a lane of every kernel, by source."""
    out = tmp_path_factory.mktemp("asm")
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        texts = pool.map(lambda s: _assembly(s, out / (s + ".s")), SOURCES)
        return {s: {name: int(size) for name, size in KERNEL_SCRATCH.findall(t)} for s, t in zip(SOURCES, texts)}


@pytest.mark.parametrize("source", SOURCES)
def test_no_scratch(scratch, source):
    sizes = scratch[source]
    assert sizes  # the kernels were found
    assert not {n: s for n, s in sizes.items() if s}
