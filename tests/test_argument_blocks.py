"""CPU: the argument blocks that the Python front end packs in one go have the layout of the structures they stand for, and the
entry points still refuse another structure."""
import ctypes

import pytest

from segquant_b200 import _lib as L
from segquant_b200 import ops


def _leaves(struct):
    """[(name, format letter, count)] of a structure's fields."""
    letters = {ctypes.c_void_p: "P", ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_float: "f", ctypes.c_double: "d"}
    out = []
    for name, kind in struct._fields_:
        if kind in letters:
            out.append((name, letters[kind], 1))
        else:
            out.append((name, letters[kind._type_], kind._length_))
    return out


def _values(letter, at):
    return at + 0.5 if letter in "fd" else at


@pytest.mark.parametrize("block,struct", [("_GEMM", L.GemmArgs), ("_ATTENTION", L.AttentionArgs), ("_ROTARY", L.RotaryArgs)])
def test_every_field_lands_in_its_place(block, struct):
    """Packs a value of its own into every field and reads it back by name; arrays of int32 travel as bytes."""
    packer = getattr(ops, block)
    args, want, at = [], {}, 1
    for name, letter, count in _leaves(struct):
        vals = [_values(letter, at + i) for i in range(count)]
        at += count
        want[name] = vals
        if count > 1 and letter == "i":
            args.append(b"".join(v.to_bytes(4, "little") for v in vals))
        else:
            args += vals
    got = struct.from_buffer_copy(packer.pack(*args))
    for name, letter, count in _leaves(struct):
        value = getattr(got, name)
        assert (list(value) if count > 1 else [value]) == want[name], name


@pytest.mark.parametrize("entry,struct", [("sq_gemm", L.GemmArgs), ("sq_attention", L.AttentionArgs), ("sq_rotary", L.RotaryArgs)])
def test_another_structure_is_refused(native_lib, entry, struct):
    fn = getattr(native_lib, entry)
    for other in (L.GatedResidualArgs(), L.NormResidual()):
        with pytest.raises(ctypes.ArgumentError):
            fn(ctypes.byref(other), None)
    with pytest.raises(ctypes.ArgumentError):
        fn(b"\0" * ctypes.sizeof(struct), None)
    assert fn(None, None) == L.SQ_ERR_INVALID_ARG and fn(ctypes.byref(struct()), None) <= 0       # its own is taken
