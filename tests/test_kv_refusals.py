"""Refusals of the cache's entry points beside those of tests/test_kv_plan.py; none of the
calls reaches a device."""
import pytest

from gollama_b200._lib import KVBatchC
from tests.test_kv_plan import APPEND, ATTEND, INVALID, READ, P, call, host, refused  # noqa: F401


@pytest.mark.parametrize("name,base", [("glc_kv_append", APPEND), ("glc_kv_read", READ), ("glc_attention_kv", ATTEND)])
@pytest.mark.parametrize("field", ["page_table", "lens", "starts"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_whole_numbers_that_are_not_aligned(call, name, base, field, off):  # noqa: F811
    batch = KVBatchC(page_table=P, lens=P, starts=P, num_seqs=4, max_pages=8, num_rows=4)
    setattr(batch, field, P + off)
    refused(call, name, base, "batch", batch, INVALID)


def test_attention_in_place_of_another_stride(call):  # noqa: F811
    """A row written would be another one's query."""
    for ld, o_ld in ((256, 260), (260, 256), (512, 1024)):
        refused(call, "glc_attention_kv", {**ATTEND, "q_ld": ld}, "o_ld", o_ld, INVALID)
