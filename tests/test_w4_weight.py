"""W4Weight made from records directly: what does not describe a weight is refused before a kernel reads past its end."""
import pytest
import torch

from micro_vllm_b200.w4_linear import W4Weight, pack_w4
from tests.w4_reference import checkpoint


@pytest.mark.parametrize('group,zeros', [(32, True), (64, False), (128, True)])
def test_records_that_do_not_describe_the_weight_are_refused(group, zeros):
    codes, scales, zero = checkpoint(130, 333, group, zeros, torch.float16, seed=1)
    weight = pack_w4(codes, scales, zero, group_size=group)
    records, shape = weight.records, weight.shape
    good = dict(records=records, shape=shape, group_size=group, has_zeros=zeros, scale_dtype=torch.float16)
    assert torch.equal(W4Weight(**good).records, records)
    assert W4Weight(**{**good, 'records': records.view(-1)}).nbytes == weight.nbytes
    for changes, message in [
        (dict(records=records[:-1]), 'bytes'),
        (dict(records=records.repeat(2, 1, 1)), 'bytes'),
        (dict(records=records.view(torch.int8)), 'uint8'),
        (dict(records=records.transpose(0, 1)), 'contiguous'),
        (dict(shape=(193, 333)), 'bytes'),
        (dict(shape=(130, 385)), 'bytes'),
        (dict(shape=(0, 333)), 'positive'),
        (dict(shape=(130,)), 'positive'),
        (dict(has_zeros=not zeros), 'bytes'),
        (dict(group_size=48), 'group_size'),
        (dict(scale_dtype=torch.float32), 'scale_dtype'),
    ]:
        with pytest.raises(RuntimeError, match=message):
            W4Weight(**{**good, **changes})
