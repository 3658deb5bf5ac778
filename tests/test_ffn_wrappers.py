"""What the Python wrappers of the feed-forward products make of tensors: every operand's device and element type is looked at,
whichever stream is passed.  (No GPU: calls that pass go on to fail the library's check of a zero dimension.)"""
import pytest
import torch

import clblas_amd as cb

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8


class Fake:
    """Stands for a tensor on a GPU."""

    def __init__(self, dtype, device=0):
        self.dtype, self.index, self.device = dtype, device, torch.device("cuda", device)

    def get_device(self):
        return self.index

    def data_ptr(self):
        return 0x1000


class FakeStream:
    cuda_stream = 0

    def __init__(self, device):
        self.device = torch.device("cuda", device)


@pytest.fixture(autouse=True)
def one_device(monkeypatch):
    cb.quantize_rows(cb.Type.F32, 0, 4, 0x1000, 0, 4, 0x1000, 0, 4, 0x1000, stream=0)  # (the wrappers look torch's names up once)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(cb, "_current_device", lambda: 0, raising=False)
    monkeypatch.setattr(cb, "_raw_stream", lambda device: 0)


def quantize_rows(t, m, **kw):
    return cb.quantize_rows(t, 0, 4, m[0], 0, 4, m[1], 0, 4, m[2], **kw)


def i8gemm(t, m, **kw):
    return cb.i8gemm(t, 0, 4, 4, m[0], 0, 4, m[1], m[2], 0, 4, m[3], m[4], 0, 4, **kw)


def gated(t, m, **kw):
    return cb.gated(t, cb.Gate.Silu, 0, 4, 4, *sum(((x, 0, 4) for x in m), ()), **kw)


def gated_i8(t, m, **kw):
    return cb.gated_i8(t, cb.Gate.Silu, 0, 4, 4, m[0], 0, 4, m[1], m[2], 0, 4, m[3], m[4], 0, 4, m[5], m[6], 0, 4, **kw)


def gated_grad(t, m, **kw):
    return cb.gated_grad(t, cb.Gate.Silu, 0, 4, 4, *sum(((x, 0, 4) for x in m), ()), **kw)


CALLS = [(quantize_rows, cb.Type.F32, [F32, I8, F32]), (quantize_rows, cb.Type.BF16, [BF16, I8, F32]), (i8gemm, cb.Type.F16, [I8, F32, I8, F32, F16]),
         (gated, cb.Type.BF16, [BF16] * 6), (gated_i8, cb.Type.F32, [I8, F32, I8, F32, I8, F32, F32]), (gated_grad, cb.Type.F16, [F16] * 9)]
IDS = ["%s-%s" % (f.__name__, t.name) for f, t, _ in CALLS]
STREAMS = [dict(), dict(stream=0), dict(stream=FakeStream(0))]


@pytest.mark.parametrize("fn,type_,dtypes", CALLS, ids=IDS)
@pytest.mark.parametrize("kw", STREAMS, ids=["current", "handle", "object"])
def test_every_operand_is_looked_at(fn, type_, dtypes, kw):
    def mats(at=None, other=None):
        return [other if i == at else Fake(d) for i, d in enumerate(dtypes)]

    assert fn(type_, mats(), **kw) == cb.Status.InvalidDim
    for i, d in enumerate(dtypes):
        for other in (Fake(d, device=1), torch.zeros(4, 4, dtype=d)):  # on another GPU; on the host
            with pytest.raises(ValueError, match="current device"):
                fn(type_, mats(i, other), **kw)
        for wrong in {F32, F16, BF16, I8, torch.float64, torch.complex64, torch.int64, torch.int32} - {d}:
            if not wrong.is_floating_point and not wrong.is_complex and wrong.itemsize == d.itemsize:
                continue
            with pytest.raises(ValueError, match="where the call takes"):
                fn(type_, mats(i, Fake(wrong)), **kw)
        raw = {4: torch.int32, 2: torch.int16, 1: torch.uint8}[d.itemsize]  # raw storage
        assert fn(type_, mats(i, Fake(raw)), **kw) == cb.Status.InvalidDim
        assert fn(type_, mats(i, 0x1000), **kw) == cb.Status.InvalidDim  # an address


@pytest.mark.parametrize("fn,type_,dtypes", CALLS, ids=IDS)
def test_all_operands_of_another_device_or_its_stream(fn, type_, dtypes):
    with pytest.raises(ValueError, match="cuda:0"):
        fn(type_, [Fake(d, device=1) for d in dtypes])
    with pytest.raises(ValueError, match="stream"):
        fn(type_, [Fake(d) for d in dtypes], stream=FakeStream(1))


def test_types_that_a_call_does_not_take_are_the_librarys_to_refuse():
    assert gated(cb.Type.F32, [Fake(F32)] * 6, stream=0) == cb.Status.InvalidValue
    assert gated_grad(7, [Fake(F16)] * 9, stream=0) == cb.Status.InvalidValue
    assert quantize_rows(9, [Fake(F32), Fake(I8), Fake(F32)], stream=0) == cb.Status.InvalidValue
