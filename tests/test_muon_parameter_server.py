"""Muon with variables and momenta on a parameter server."""
import pytest


def test_a_counter_on_the_parameter_server_is_shipped_by_a_gpu_worker():
    """Muon's step counter is an ``AssignAdd`` of its own (matrices and vectors are two nodes): the
    GPU kernel of the op hands variables of another process to their store."""
    import types

    import torch

    from distributed_tensorflow_amd.framework.op_registry import get_opdef
    from distributed_tensorflow_amd.ops import hip_kernels  # noqa: F401
    from distributed_tensorflow_amd.parallel.ps_transport import RemoteVariableStore
    store = object.__new__(RemoteVariableStore)        # (no connection: nothing is sent here)
    shipped = []
    ctx = types.SimpleNamespace(
        session=types.SimpleNamespace(_store_for=lambda op: store),
        var_assign_add=lambda op, delta: shipped.append((op.name, float(delta))),
        note_fallback=lambda op, why: pytest.fail("refused: %s" % why))
    var = types.SimpleNamespace(name="global_step")
    for kind, sign in (("AssignAdd", 1.0), ("AssignSub", -1.0)):
        op = types.SimpleNamespace(name="add", type=kind, inputs=[types.SimpleNamespace(op=var)])
        get_opdef(kind).hip_kernel(op, [None, torch.tensor(3.0)], ctx)
        assert shipped.pop() == ("global_step", 3.0 * sign)
