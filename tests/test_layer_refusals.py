"""CPU tests of calls around a decoder layer's products that share memory or pass a limit:
refused before any device call."""
import pytest

from gollek_amd import tensor_ops as ops
from tests.test_layer_ops import BASE, BF16, append, attend, cache


@pytest.mark.parametrize("name", ["k_ptr", "v_ptr"])
def test_append_of_keys_or_values_that_its_query_results_overwrite(name):
    # queries in place, and the keys (or values) at their address as well: as large, of the same stride
    q = BASE + (8 << 20)
    with pytest.raises(ops.IllegalArgumentError, match="overlaps the " + ("keys" if name == "k_ptr" else "values")):
        append(cache(), type_id=BF16, q_heads=2, q_ptr=q, q_out_ptr=q, **{name: q})


@pytest.mark.parametrize("kw,name", [(dict(page_table_ptr=BASE + (4 << 20), max_pages=100), "page table"),
                                     (dict(lengths_ptr=BASE + (4 << 20), sequences=200), "lengths")])
def test_attention_whose_results_lie_in_what_starts_at_its_queries(kw, name):
    # results between the queries' rows are fine, but not over another input at the queries' address
    q = BASE + (4 << 20)
    with pytest.raises(ops.IllegalArgumentError, match="output overlaps the " + name):
        attend(cache(), **{**dict(q_ptr=q, q_stride=512, out_ptr=q + 512, out_type=BF16, out_stride=512), **kw})
