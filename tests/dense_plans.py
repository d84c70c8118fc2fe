"""Which kernel a projection of given sizes takes (``moe_linear_query``): tests that are about one kernel assert that they
reach it, so that a change of the rules cannot leave it untested unnoticed."""
import ctypes


def plan(m, n, k, gated=False, **kw):
    """The plan as a dict, ``kernel`` by name; of a call on aligned, contiguous tensors unless ``kw`` says otherwise."""
    from nano_ktrans_b200 import _lib

    # addresses far apart that nothing reads: the query only looks at them
    d = dict(x_dev=1 << 40, w_dev=1 << 41, w_up_dev=1 << 42 if gated else None, bias_dev=None, residual_dev=None,
             out_dev=1 << 43, ldx=k, ldw=k, ldw_up=k, ldr=n, ldo=n, m=m, n=n, k=k, dtype=0, activation=0)
    d.update(kw)
    out, err = _lib.MoeLinearPlan(), ctypes.create_string_buffer(256)
    rc = _lib.lib().moe_linear_query(ctypes.byref(_lib.MoeLinearDesc(**d)), ctypes.byref(out), err, len(err))
    assert rc == _lib.MOE_OK, err.value
    p = {name: getattr(out, name) for name, _ in out._fields_}
    return dict(p, kernel=_lib.LINEAR_KERNELS[p["kernel"]])


def kernel(m, n, k, gated=False, **kw):
    return plan(m, n, k, gated, **kw)["kernel"]
