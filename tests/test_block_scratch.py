"""Generated code: the kernels of layer norm, linear and clipping keep to their registers.

The exceptions are named: the FP32 norm backward with eight vectors a lane (8193 to 16384 columns)
spills some of its own, beside the sums for the parameters.
"""

from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_store_hazard import KERNEL_SCRATCH, _assembly

SOURCES = ("layer_norm.hip", "linear.hip", "linear_product.hip", "linear_wide.hip", "linear_narrow.hip",
           "linear_f32.hip", "grad_clip.hip")  # fmt: skip
SPILLING = tuple(f"norm_bwd_kernelINS_3F32ELb{whole}ELi8ELi8ELb1E" for whole in (0, 1))


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
    assert not {n: s for n, s in sizes.items() if s and not any(k in n for k in SPILLING)}
