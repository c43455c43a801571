"""CPU: which layers of a step have their new rows (fpga_qwen_b200/paged.py: StepOrder)."""
import pytest

from fpga_qwen_b200.paged import StepOrder
from fpga_qwen_b200.qattn import QA_ERR_STATE, QAttnError


def refused(call):
    with pytest.raises(QAttnError) as err:
        call()
    assert err.value.status == QA_ERR_STATE


def test_a_step_ends_with_the_last_layers_rows():
    s = StepOrder(3)
    s.check_complete("evict")
    s.check_written(0, 3)                               # no step: rows of earlier steps
    s.begin([0, 2])
    refused(lambda: s.check_complete("evict"))
    refused(lambda: s.check_written(0, 1))
    s.wrote(1, 1)
    s.check_written(1, 1)
    refused(lambda: s.check_written(0, 2))
    refused(lambda: s.check_complete("evict"))
    s.wrote(0, 1)
    s.wrote(0, 1)                                       # again: the same rows
    s.check_written(0, 2)
    refused(lambda: s.check_written(0, 3))
    s.wrote(2, 1)
    s.check_complete("evict")
    s.begin([0])
    s.wrote(0, 3)
    s.check_complete("begin_step")


def test_a_step_without_sequences_is_over():
    s = StepOrder(2)
    s.begin([0, 1])
    s.close(2)
    s.close(0)
    refused(lambda: s.check_complete("evict"))
    s.close(1)
    s.check_complete("evict")
    s.check_written(0, 2)
    s.begin([1])
    refused(lambda: s.check_complete("evict"))


def test_captured_appends_end_the_watch():
    s = StepOrder(2)
    s.begin([0])
    s.captured()
    s.check_complete("evict")
    s.begin([0])
    s.check_complete("begin_step")
    s.check_written(0, 2)
