"""Arguments that the operators around the projections refuse before any device work (no GPU needed): adapters, norms around the
residual sum, verification of drafted tokens."""
import ctypes

import numpy as np
import pytest

import overfit_amd as ov
from overfit_amd import _lib

F = np.float32


class FakeWeight:
    InputSize, OutputSize, context = 64, 8, None


@pytest.mark.parametrize("args,error", [
    ((0, 8, 4, 4), ov.OverfitArgumentOutOfRangeError),
    ((64, 0, 4, 4), ov.OverfitArgumentOutOfRangeError),
    ((48, 8, 4, 4), ov.OverfitArgumentError),  # not a multiple of 32
    ((64, 8, 0, 4), ov.OverfitArgumentOutOfRangeError),
    ((64, 8, 4097, 4), ov.OverfitArgumentOutOfRangeError),
    ((64, 8, 4, 0), ov.OverfitArgumentOutOfRangeError),
    ((64, 8, 4, 257), ov.OverfitArgumentOutOfRangeError),
    ((64, 8, 4, 4, 12), ov.OverfitUnsupportedTypeError),  # a block type
])
def test_adapter_set_sizes(args, error):
    with pytest.raises(error):
        ov.AdapterSet(*args)


def loose_set(input_size=64, output_size=8, slots=2, max_rank=4, type_id=ov.TYPE_F16):
    s = ov.AdapterSet.__new__(ov.AdapterSet)  # no device: only what load() checks before it calls the library
    s.input_size, s.output_size, s.slots, s.max_rank, s.type_id = input_size, output_size, slots, max_rank, type_id
    return s


@pytest.mark.parametrize("slot,a,b,error", [
    (-1, (4, 64), (8, 4), ov.OverfitArgumentOutOfRangeError),
    (2, (4, 64), (8, 4), ov.OverfitArgumentOutOfRangeError),
    (0, (5, 64), (8, 5), ov.OverfitArgumentOutOfRangeError),  # above max_rank
    (0, (0, 64), (8, 0), ov.OverfitArgumentOutOfRangeError),
    (0, (4, 63), (8, 4), ov.OverfitArgumentError),
    (0, (4, 64), (7, 4), ov.OverfitArgumentError),
    (0, (4, 64), (8, 3), ov.OverfitArgumentError),
    (0, (64,), (8, 4), ov.OverfitArgumentError),
])
def test_adapter_load_shapes(slot, a, b, error):
    with pytest.raises(error):
        loose_set().load(slot, np.zeros(a, np.float16), np.zeros(b, np.float16))


def test_adapter_load_types():
    s = loose_set()
    with pytest.raises(ov.OverfitArgumentNullError):
        s.load(0, None, np.zeros((8, 4), np.float16))
    with pytest.raises(ov.OverfitArgumentError):
        s.load(0, np.zeros((4, 64), F), np.zeros((8, 4), np.float16))
    with pytest.raises(ov.OverfitArgumentError):
        s.load(0, np.zeros((64, 4), np.float16).T, np.zeros((8, 4), np.float16))  # a transposed view
    with pytest.raises(ov.OverfitArgumentOutOfRangeError):
        s.unload(2)


@pytest.mark.parametrize("change,error", [
    (dict(weights=[]), ov.OverfitArgumentOutOfRangeError),
    (dict(weights=[FakeWeight()] * 5, adapters=[None] * 5), ov.OverfitArgumentOutOfRangeError),
    (dict(adapters=[]), ov.OverfitArgumentError),
    (dict(rows=0), ov.OverfitArgumentOutOfRangeError),
    (dict(x=np.zeros(127, F)), ov.OverfitArgumentError),
    (dict(x=np.zeros(128, np.float64)), ov.OverfitArgumentError),
    (dict(row_slots=np.zeros(1, np.int32)), ov.OverfitArgumentError),
    (dict(row_slots=np.zeros(2, np.int64)), ov.OverfitArgumentError),
    (dict(row_slots=None), ov.OverfitArgumentNullError),
    (dict(outs=[np.zeros(15, F)]), ov.OverfitArgumentError),
    (dict(outs=[]), ov.OverfitArgumentError),
    (dict(biases=[np.zeros(7, F)]), ov.OverfitArgumentError),
])
def test_project_adapters_arguments(change, error):
    call = dict(weights=[FakeWeight()], adapters=[None], x=np.zeros(128, F), row_slots=np.zeros(2, np.int32), rows=2)
    call.update(change)
    with pytest.raises(error):
        ov.project_adapters(**call)


@pytest.mark.parametrize("change,error", [
    (dict(y=None), ov.OverfitArgumentNullError),
    (dict(y=np.zeros(0, F)), ov.OverfitArgumentError),
    (dict(rows=0), ov.OverfitArgumentOutOfRangeError),
    (dict(rows=5), ov.OverfitArgumentError),  # 64 values are no five rows
    (dict(gate=np.zeros(16, F)), ov.OverfitArgumentError),  # no axis
    (dict(gate_axis="channel"), ov.OverfitArgumentError),  # no gate
    (dict(gate=np.zeros(16, F), gate_axis="column"), ov.OverfitArgumentError),
    (dict(gate=np.zeros(15, F), gate_axis="channel"), ov.OverfitArgumentError),
    (dict(gate=np.zeros(3, F), gate_axis="row"), ov.OverfitArgumentError),
    (dict(gate=np.zeros(63, F), gate_axis="full"), ov.OverfitArgumentError),
    (dict(residual=np.zeros(63, F)), ov.OverfitArgumentError),
    (dict(x_out=np.zeros(64, F)), ov.OverfitArgumentError),  # no pre norm
    (dict(pre=ov.Norm(np.zeros(15, F))), ov.OverfitArgumentError),
    (dict(post=ov.Norm(bias=np.zeros(15, F))), ov.OverfitArgumentError),
    (dict(pre="rms"), ov.OverfitArgumentError),
    (dict(pre=ov.Norm(), x_out=np.zeros(63, F)), ov.OverfitArgumentError),
    (dict(h_out=np.zeros(63, F)), ov.OverfitArgumentError),
    (dict(y=np.zeros((16, 4), F).T), ov.OverfitArgumentError),  # not contiguous
])
def test_residual_norm_arguments(change, error):
    call = dict(y=np.zeros(64, F), rows=4)
    call.update(change)
    with pytest.raises(error):
        ov.residual_norm(**call)


def test_norm_arguments():
    with pytest.raises(ov.OverfitArgumentError):
        ov.Norm(kind="batch")
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ov.OverfitArgumentOutOfRangeError):
            ov.Norm(eps=eps)


@pytest.mark.parametrize("change,error", [
    (dict(vocab=0), ov.OverfitArgumentOutOfRangeError),
    (dict(vocab=9), ov.OverfitArgumentError),
    (dict(logits=np.zeros(0, F)), ov.OverfitArgumentError),
    (dict(row_offsets=np.zeros(1, np.int32)), ov.OverfitArgumentError),
    (dict(row_offsets=np.zeros(6, np.int32)), ov.OverfitArgumentError),  # five requests in four rows
    (dict(row_offsets=np.zeros(2, np.int64)), ov.OverfitArgumentError),
    (dict(draft_tokens=np.zeros(2, np.int32)), ov.OverfitArgumentError),
    (dict(draft_tokens=None), ov.OverfitArgumentNullError),
    (dict(accept_uniforms=np.zeros(2, F)), ov.OverfitArgumentError),
    (dict(final_uniforms=np.zeros(0, F)), ov.OverfitArgumentError),
    (dict(draft_probs=np.zeros(29, F)), ov.OverfitArgumentError),
    (dict(temperature=np.zeros(0, F)), ov.OverfitArgumentError),
    (dict(accepted=np.zeros(0, np.int32)), ov.OverfitArgumentError),
    (dict(tokens=np.zeros(3, np.int32)), ov.OverfitArgumentError),
])
def test_verify_drafts_arguments(change, error):
    call = dict(logits=np.zeros(40, F), vocab=10, row_offsets=np.array([0, 4], np.int32),
                draft_tokens=np.zeros(3, np.int32), accept_uniforms=np.zeros(3, F), final_uniforms=np.zeros(1, F))
    call.update(change)
    with pytest.raises(error):
        ov.verify_drafts(**call)


def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    h = ctypes.c_void_p()
    assert lib.ovfq_adapters_create(None, 1, 64, 8, 1, 4, ctypes.byref(h)) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_adapters_destroy(None) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_adapters_load(None, 0, None, None, 1, 1.0) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_adapters_unload(None, 0) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_adapters_info(None, None, None, None, None, None, None) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_project_adapters_dev(None, 1, None, None, None, 1, None, None, None) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_residual_norm_dev(None, None, None, 1, 8, None, None, 0, 1.0, None, None, None) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_verify_drafts_dev(*[None] * 2, 1, 8, 1, *[None] * 8) == _lib.OVFQ_ERR_NULL
