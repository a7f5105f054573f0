"""What the kernels of the paged cache's small calls ask the hardware for: no
private memory, whose set-up a launch of some 10 us would pay for."""
import pytest

from tests import code_object

pytestmark = pytest.mark.skipif(not code_object.available(), reason="library not built, or no ROCm tools")


@pytest.mark.parametrize("params", ["PagedFattnParams", "PagedWindowParams", "PagedTreeParams", "PagedSeesParams"])
def test_attention_over_the_paged_cache_has_no_private_memory(params):
    sizes = {n: k["private_segment_fixed_size"] for n, k in code_object.kernels().items()
             if params in n and ("paged_fattn_kernel" in n or "paged_join_kernel" in n)}
    assert len(sizes) == 7 and not any(sizes.values()), sizes
