"""An earlier call's failure is none of the one-call operators' on the GPU: a
refused allocation leaves an error on the thread, which a launch's check must
not take for its own."""

import numpy as np
import pytest

import mx4_cases as M
from attention_cases import CASES, inputs, oracle
from furykernel_amd import mx4, paged, runtime
from test_gpu_ops import run_op
from test_gpu_serve import attend_inputs, bind_attend, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def refuse(device):
    with pytest.raises(runtime.FkError) as err:
        device.alloc(1 << 50)
    assert err.value.status == -6, err.value       # out of device memory


def test_a_refused_allocation_is_not_the_next_operators_error(device, mem):
    x = attend_inputs(np.random.default_rng(1), [40, 300], 4, 2, 64, 16, "f16")
    attend, read, _ = bind_attend(device, mem, x, 0.125)
    attend.enqueue()
    device.sync()
    want = read()
    sizes = dict(cached=2, fresh=2, free=4, head=1, table=4, lengths=2, starts=3, slots=2, positions=2, owner=2,
                 counts=4)
    words = {name: mem.empty(4 * n) for name, n in sizes.items()}
    for name, values in dict(cached=[3, 0], fresh=[1, 1], free=[5, 6, 7, 8], head=[0], table=[4, 0, 0, 0]).items():
        words[name].write(np.uint32(values))
    plan = paged.PagePlan(device, **words, requests=2, tokens=2, table_len=2, block_size=16, free_len=4)
    rows = np.random.default_rng(2).standard_normal((5, 40)).astype(np.float32)
    held = mem.keep(mx4.Mx4Matrix(device, 5, 40))
    quantize = mx4.Quantize(device, mem.put(rows), held)
    for op in (plan, quantize, attend):
        refuse(device)
        op.enqueue()
    device.sync()
    assert np.array_equal(read(), want)
    assert words["slots"].read(np.uint32, 2).tolist() == [4 * 16 + 3, 5 * 16]
    assert np.array_equal(held.codes.read(np.uint8), M.pack(*M.quantize(rows))[0])


def test_a_refused_allocation_is_not_the_decode_attentions_error(device):
    x = inputs(CASES[4])
    run_op(device, x)                              # (the workspace as large as the next call needs)
    call = runtime.attend_decode

    def after_a_refusal(dev, args, **kw):
        refuse(dev)
        call(dev, args, **kw)

    runtime.attend_decode = after_a_refusal
    try:
        out = run_op(device, x)[2]
    finally:
        runtime.attend_decode = call
    assert np.array_equal(out.view(np.uint32), oracle(x)["out"].view(np.uint32))
