"""Host-side checks of the operators around a training step's products -- no GPU needed: what their C
entry points refuse, with which status and message, before anything is launched.  Addresses are
stand-ins and never dereferenced."""

import ctypes

import pytest

from flash_train import capi as c

FAKE = 0x7F0000000000  # aligned stand-in device address
BIG = 1 << 62


def view(dims, kind=c.FP32, memory=FAKE, host=False, strides=None):
    index = c.INDEX_INVALID if strides is not None else c.INDEX_CONTINUOUS
    return c.View(memory, dims, numeric_type=kind, index_type=index, host=host, strides=strides)


def fails(status, text, call, *args):
    lib = c.lib()
    args = [a.sv if isinstance(a, c.View) else a for a in args]
    assert getattr(lib, call)(*args) == status, c.last_message()
    message = c.last_message()
    assert message.startswith(call + ": ") or text.startswith("StorageView"), message
    assert text in message, message


def head(**changed):
    t, h, v = 6, 16, 20
    views = {"hidden": view([t, h]), "weight": view([v, h]), "target": view([t], c.INT64), "loss": view([t]),
             "lse": view([t]), "ignore": -100, "workspace": FAKE, "bytes": BIG, "stream": None}
    views.update(changed)
    return list(views.values())


@pytest.mark.parametrize("status,text,changed", [
    (c.INVALID_ARGUMENT, "hidden must be in device memory", {"hidden": view([6, 16], host=True)}),
    (c.INVALID_ARGUMENT, "hidden must have rank 2, got 1", {"hidden": view([6])}),
    (c.INVALID_ARGUMENT, "hidden must not be null", {"hidden": view([6, 16], memory=None)}),
    (c.INVALID_ARGUMENT, "hidden has 16 columns, weight 8", {"weight": view([20, 8])}),
    (c.INVALID_ARGUMENT, "at least one class", {"weight": view([0, 16])}),
    (c.UNSUPPORTED, "must be fp32, bf16 or fp16", {"hidden": view([6, 16], c.FP64)}),
    (c.UNSUPPORTED, "one numeric type", {"weight": view([20, 16], c.BF16)}),
    (c.UNSUPPORTED, "contiguous rows", {"hidden": view([6, 16], strides=[1, 6])}),
    (c.UNSUPPORTED, "rows that overlap", {"weight": view([20, 16], strides=[8, 1])}),
    (c.UNSUPPORTED, "not aligned", {"hidden": view([6, 16], memory=FAKE + 2)}),
    (c.UNSUPPORTED, "row stride go to", {"weight": view([20, 16], strides=[(1 << 20) + 1, 1])}),
    (c.UNSUPPORTED, "tokens and classes", {"weight": view([1 << 31, 16])}),
    (c.UNSUPPORTED, "target has numeric type", {"target": view([6])}),
    (c.INVALID_ARGUMENT, "target has size 5", {"target": view([5], c.INT32)}),
    (c.UNSUPPORTED, "target must be dense", {"target": view([6], c.INT32, strides=[2])}),
    (c.UNSUPPORTED, "loss has numeric type", {"loss": view([6], c.BF16)}),
    (c.INVALID_ARGUMENT, "lse must not be null", {"lse": view([6], memory=None)}),
    (c.INVALID_ARGUMENT, "the workspace holds 0 bytes", {"bytes": 0}),
    (c.INVALID_ARGUMENT, "the workspace holds", {"workspace": None}),
    (c.INVALID_ARGUMENT, "aligned to 256 bytes", {"workspace": FAKE + 16}),
])
def test_cross_entropy_refuses(status, text, changed):
    fails(status, text, "ftrainLinearCrossEntropy", *head(**changed))


def test_cross_entropy_backward_refuses():
    def call(**changed):
        views = {"grad_loss": view([6]), "hidden": view([6, 16]), "weight": view([20, 16]), "target": view([6], c.INT32),
                 "lse": view([6]), "grad_hidden": view([6, 16]), "grad_weight": view([20, 16]), "ignore": -100,
                 "workspace": FAKE, "bytes": BIG, "stream": None}
        views.update(changed)
        return list(views.values())

    name = "ftrainLinearCrossEntropyBackward"
    fails(c.INVALID_ARGUMENT, "grad_loss has size 3", name, *call(grad_loss=view([3])))
    fails(c.INVALID_ARGUMENT, "grad_hidden must be 6 x 16", name, *call(grad_hidden=view([6, 15])))
    fails(c.UNSUPPORTED, "grad_weight has numeric type", name, *call(grad_weight=view([20, 16], c.FP16)))
    fails(c.UNSUPPORTED, "grad_weight has rows that overlap", name, *call(grad_weight=view([20, 16], strides=[4, 1])))
    fails(c.INVALID_ARGUMENT, "the workspace holds 16 bytes", name, *call(bytes=16))


def test_cross_entropy_workspace_does_not_hold_the_logits():
    """Two million classes: the workspace stays a fraction of the logits' bytes."""
    n = ctypes.c_uint64()
    for backward in (False, True):
        for kind, size in ((c.FP32, 4), (c.BF16, 2)):
            args = view([4096, 1024], kind).sv, view([1 << 21, 1024], kind).sv
            assert c.lib().ftrainLinearCrossEntropyWorkspaceBytes(*args, backward, ctypes.byref(n)) == c.SUCCESS
            assert 4096 * 1024 * size < n.value < 4096 * (1 << 21) * size // 4
    fails(c.INVALID_ARGUMENT, "output must not be null", "ftrainLinearCrossEntropyWorkspaceBytes", view([4, 8]), view([9, 8]),
          True, None)


def route(**changed):
    t, n, k = 6, 8, 2
    views = {"logits": view([t, n]), "mask": view([t], c.UINT8, memory=None), "experts": view([t, k], c.INT32),
             "gates": view([t, k]), "slots": view([t, k], c.INT32), "counts": view([n], c.INT32),
             "routed": view([1], c.INT32), "loss": view([1]), "normalize": True, "workspace": FAKE, "bytes": BIG,
             "stream": None}
    views.update(changed)
    return list(views.values())


@pytest.mark.parametrize("status,text,changed", [
    (c.UNSUPPORTED, "1 to 1024 experts", {"logits": view([6, 1025])}),
    (c.UNSUPPORTED, "1 to 1024 experts", {"logits": view([6, 0])}),
    (c.UNSUPPORTED, "1 to 32 of its experts, got 9 of 8", {"experts": view([6, 9], c.INT32)}),
    (c.UNSUPPORTED, "1 to 32 of its experts, got 0 of 8", {"experts": view([6, 0], c.INT32)}),
    (c.UNSUPPORTED, "choices are supported", {"logits": view([1 << 30, 8]), "experts": view([1 << 30, 2], c.INT32)}),
    (c.UNSUPPORTED, "experts has numeric type", {"experts": view([6, 2], c.INT64)}),
    (c.INVALID_ARGUMENT, "experts has size 5", {"experts": view([5, 2], c.INT32)}),
    (c.UNSUPPORTED, "mask has numeric type", {"mask": view([6], c.FP32)}),
    (c.INVALID_ARGUMENT, "mask has size 7", {"mask": view([7], c.UINT8)}),
    (c.INVALID_ARGUMENT, "gates has size 3 in dimension 1", {"gates": view([6, 3])}),
    (c.INVALID_ARGUMENT, "counts has size 7", {"counts": view([7], c.INT32)}),
    (c.UNSUPPORTED, "slots must be dense", {"slots": view([6, 2], c.INT32, strides=[4, 1])}),
    (c.INVALID_ARGUMENT, "balance_loss must not be null", {"loss": view([1], memory=None)}),
    (c.INVALID_ARGUMENT, "the workspace holds 100 bytes", {"bytes": 100}),
])
def test_route_refuses(status, text, changed):
    fails(status, text, "ftrainMoeRoute", *route(**changed))


def test_route_backward_refuses():
    good = [view([6, 2]), view([1]), view([6, 8]), view([6], c.UINT8, memory=None), view([6, 2], c.INT32),
            view([8], c.INT32), view([1], c.INT32), view([6, 8]), False, None]
    for i, bad, status, text in ((0, view([6, 1]), c.INVALID_ARGUMENT, "grad_gates has size 1"),
                                 (1, view([2]), c.INVALID_ARGUMENT, "grad_loss has size 2"),
                                 (7, view([6, 9]), c.INVALID_ARGUMENT, "grad_logits must be 6 x 8"),
                                 (7, view([6, 8], c.BF16), c.UNSUPPORTED, "grad_logits has numeric type")):
        args = list(good)
        args[i] = bad
        fails(status, text, "ftrainMoeRouteBackward", *args)


def test_clip_refuses():
    def array(*views):
        return (c.StorageView * len(views))(*[v.sv for v in views])

    norm, name = view([1]), "ftrainClipGradNorm"
    grads = array(view([4]), view([3, 2], c.BF16))

    def bad(status, text, g=grads, out=None, n=2, norm=norm, most=1.0, eps=0.0, workspace=FAKE, size=BIG):
        fails(status, text, name, g, out, n, norm, most, eps, workspace, size, None)

    bad(c.INVALID_ARGUMENT, "grads must not be null", g=None)
    bad(c.INVALID_ARGUMENT, "must not be negative", most=-1.0)
    bad(c.INVALID_ARGUMENT, "must not be negative", most=float("nan"))
    bad(c.INVALID_ARGUMENT, "must not be negative", eps=-1.0)
    bad(c.INVALID_ARGUMENT, "grads[1] must be in device memory", g=array(view([4]), view([4], host=True)))
    bad(c.UNSUPPORTED, "grads[0] must be fp32, bf16 or fp16", g=array(view([4], c.INT32), view([4])))
    bad(c.UNSUPPORTED, "grads[0] must be continuous", g=array(view([4, 4], strides=[8, 1]), view([4])))
    bad(c.UNSUPPORTED, "grads[0] is not aligned", g=array(view([4], memory=FAKE + 1), view([4])))
    bad(c.INVALID_ARGUMENT, "grads[0] must not be null", g=array(view([4], memory=None), view([4])))
    bad(c.OVERFLOW, "too many elements", g=array(view([1 << 40, 1 << 40]), view([4])))
    bad(c.INVALID_ARGUMENT, "outputs[1] must be like grads[1]", out=array(view([4]), view([5], c.BF16)))
    bad(c.INVALID_ARGUMENT, "norm has size 2", norm=view([2]))
    bad(c.INVALID_ARGUMENT, "the workspace holds 8 bytes", size=8)
