"""Where an allocation lies on the device: the bytes there are its own, and work on the null stream is in order with
what is submitted."""
import numpy as np
import pytest
import torch

from forja_amd.core import BackendError, CommandList, DType, Op, Status
from tests.test_host_calls import fake  # noqa: F401  (the fixture)


def test_bytes_at_the_address(fake):  # noqa: F811
    """(this runtime's device memory is the host's)"""
    fake("""
t = hip.alloc(DType.F32, (4, 8))
hip.write_array(t, np.arange(32, dtype=np.float32))
assert np.frombuffer(ctypes.string_at(hip.device_address(t), 128), np.float32).tolist() == list(range(32))
assert hip.device_address(t.narrow(0, 2, 1)) == hip.device_address(t) + 64
held = hip.import_readonly(b"abcd" * 4, DType.U32, (4,))
assert ctypes.string_at(hip.device_address(held), 16) == b"abcd" * 4
hip.release(t)
try:
    hip.device_address(t)
except BackendError as e:
    assert e.status.name == "INVALID_INPUT"
else:
    raise SystemExit("an address of what is released")
assert load_library().fh_device_address(hip._handle, held.buffer, None) != 0
""")


class Shared:
    """An allocation as torch takes it."""

    def __init__(self, backend, tensor):
        self.backend, self.tensor = backend, tensor
        self.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": "<f4", "version": 2, "strides": None,
                                         "data": (backend.device_address(tensor), False)}


@pytest.mark.gpu
def test_work_on_the_null_stream_is_in_order_with_submissions(hip):
    """torch writes the input of each submission and reads its output, and nobody waits in between."""
    n, turns = 1 << 22, 20
    a, b = hip.alloc(DType.F32, (n,)), hip.alloc(DType.F32, (n,))
    at_a, at_b = (torch.as_tensor(Shared(hip, t), device="cuda") for t in (a, b))
    assert at_a.data_ptr() == hip.device_address(a) and at_b.data_ptr() == hip.device_address(b)
    commands = CommandList()
    commands.dispatch(Op.copy(), [a], b)
    seen, waiting = [], []
    for turn in range(turns):
        at_a.fill_(float(turn + 1))
        waiting.append(hip.submit(commands))
        seen.append(at_b.clone())
        at_b.zero_()
    for submission in waiting:
        submission.wait()
    for turn, values in enumerate(seen):
        assert bool((values == turn + 1).all()), turn
    torch.cuda.synchronize()
    hip.write_array(a, np.arange(n, dtype=np.float32))
    assert torch.equal(at_a, torch.arange(n, dtype=torch.float32, device="cuda"))
    with pytest.raises(BackendError) as info:
        hip.device_address(type(a)(0, a.layout, True))
    assert info.value.status == Status.INVALID_INPUT
