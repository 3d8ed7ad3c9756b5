"""The operators on device tensors, without a device: their refusals (every wrong argument is an error before the device is touched) and the argument structs' layout."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from vadc_amd import _lib, ops
from vadc_amd.engine import VadcAmdError


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_argument_structs_are_packed_as_the_header_lays_them_out(tmp_path):
    text = open(os.path.join(ROOT, "include", "vadc_amd.h")).read()
    names = {"linear": ops._LINEAR, "group_norm": ops._NORM, "gated_delta": ops._DELTA}
    src = '#include <stdio.h>\n#include "vadc_amd.h"\nint main(void) {\n'
    for n in names:
        body = re.search(r"typedef struct vadc_amd_%s_args \{(.*?)\}" % n, text, re.S).group(1)
        fields = re.findall(r"([a-z_]+)(?:\[\d\])?[,;]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
        src += f'printf("%zu", sizeof(vadc_amd_{n}_args));' + "".join(f'printf(" %zu:%zu", offsetof(vadc_amd_{n}_args, {f}), sizeof(((vadc_amd_{n}_args *)0)->{f}));' for f in fields) + 'printf("\\n");\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    for line, (n, packed) in zip(subprocess.check_output([str(tmp_path / "s")], text=True).splitlines(), names.items()):
        size, *fields = line.split()
        assert int(size) == packed.size, n
        at = 0
        for f in fields:                                             # no holes: "=" packs without padding
            offset, width = map(int, f.split(":"))
            assert offset == at, (n, f)
            at += width
        assert at == packed.size


@pytest.mark.parametrize("kw, error", [
    (dict(x=t(3, 5), weight=t(4, 6)), ValueError),
    (dict(x=t(3, 5), weight=t(5)), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), bias=t(5)), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), residual=t(3, 5)), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), out=t(4, 3)), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), activation="tanh"), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), activation=None), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5, dtype=torch.bfloat16)), TypeError),
    (dict(x=t(3, 5, dtype=torch.float64), weight=t(4, 5, dtype=torch.float64)), TypeError),
    (dict(x=t(5, 3).T, weight=t(4, 5)), ValueError),                 # the last dimension is not contiguous
    (dict(x=t(3, 5), weight=t(5, 4).T), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5).requires_grad_()), ValueError),
    (dict(x=t(3, 5), weight=t(4, 5), residual_first=t(1)), TypeError),
    (dict(x=t(3, 5), weight=t(4, 5)), ValueError),                   # no device
])
def test_linear_refuses(kw, error):
    with pytest.raises(error, match="linear"):
        ops.linear(**kw)


@pytest.mark.parametrize("kw, error", [
    (dict(x=t(8), groups=2), ValueError),
    (dict(x=t(3, 8), groups=3), ValueError),
    (dict(x=t(3, 8), groups=0), ValueError),
    (dict(x=t(3, 8), groups=2.0), TypeError),
    (dict(x=t(3, 8), groups=2, eps=t(1)), TypeError),
    (dict(x=t(3, 8), groups=2, eps=1e39), ValueError),
    (dict(x=t(3, 8), groups=2, eps=-1.0), ValueError),
    (dict(x=t(3, 8), groups=2, eps=float("nan")), ValueError),
    (dict(x=t(3, 8), groups=2, weight=t(4)), ValueError),
    (dict(x=t(3, 8), groups=2, gate=t(3, 1, 8)), ValueError),
    (dict(x=t(3, 8), groups=2, out=t(2, 8)), ValueError),
    (dict(x=t(3, 4, 8), groups=2, lengths=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(x=t(3, 4, 8), groups=2, lengths=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(x=t(3, 8), groups=2, weight=t(8, dtype=torch.float16)), TypeError),
    (dict(x=t(8, 4).T, groups=2), ValueError),
    (dict(x=t(3, 8), groups=2, activation="softmax"), ValueError),
    (dict(x=t(3, 8).requires_grad_(), groups=2), ValueError),
    (dict(x=t(3, 8), groups=2), ValueError),
])
def test_group_norm_refuses(kw, error):
    with pytest.raises(error, match="group_norm"):
        ops.group_norm(**kw)


def delta_args(b=2, steps=3, hk=1, h=2, dk=4, dv=5, **kw):
    a = dict(q=t(b, steps, hk, dk), k=t(b, steps, hk, dk), v=t(b, steps, h, dv), log_decay=t(b, steps, h), beta=t(b, steps, h), state=t(b, h, dk, dv))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, error", [
    (dict(q=t(2, 3, 4)), ValueError),
    (dict(k=t(2, 3, 1, 5)), ValueError),
    (dict(v=t(2, 4, 2, 5)), ValueError),
    (dict(hk=2, h=3), ValueError),
    (dict(dk=257), ValueError),
    (dict(beta=t(2, 3)), ValueError),
    (dict(state=t(2, 2, 5, 4)), ValueError),
    (dict(state=t(2, 2, 5, 4).transpose(2, 3)), ValueError),
    (dict(state=t(2, 2, 4, 5, dtype=torch.bfloat16)), TypeError),
    (dict(beta=t(2, 3, 2, dtype=torch.bfloat16)), TypeError),
    (dict(v=t(2, 3, 2, 5, dtype=torch.float16)), TypeError),
    (dict(out=t(2, 3, 5, 2)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(scale=t(1)), TypeError),
    (dict(normalize=t(1)), TypeError),
    (dict(scale=float("inf")), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(q=t(2, 3, 1, 8)[..., ::2]), ValueError),
    (dict(state=t(2, 2, 4, 5).requires_grad_()), ValueError),
    (dict(), ValueError),
])
def test_gated_delta_refuses(kw, error):
    with pytest.raises(error, match="gated_delta"):
        ops.gated_delta(**delta_args(**kw))


def pack(fmt, **changed):
    """a valid argument struct of small sizes at made-up addresses (nothing is read before the checks are through), with fields changed by their place"""
    fields = {
        "linear": [0x1000, 0x2000, 0, 0, 0x3000, 2, 8, 8, 8, 8, 8, 8, 0, 0, 0, -1],
        "group_norm": [0x1000, 0, 0, 0, 0x3000, 0, 0, 0, 2, 3, 8, 2, 24, 8, 24, 8, 24, 8, 0, 0, -1, 1e-5],
        "gated_delta": [0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 0, 0, 0, 2, 1, 1, 2, 4, 8] + [4, 4, 4] * 2 + [16, 16, 8] * 2 + [2, 2, 2, 2, 64, 1.0, 0, 0, -1],
    }[fmt]
    for at, value in changed.items():
        fields[int(at[1:])] = value
    return {"linear": ops._LINEAR, "group_norm": ops._NORM, "gated_delta": ops._DELTA}[fmt].pack(*fields)


@pytest.mark.parametrize("op, changed", [
    ("linear", dict(_0=0)), ("linear", dict(_4=0)), ("linear", dict(_0=0x1001)), ("linear", dict(_5=-1)), ("linear", dict(_5=2 ** 41)), ("linear", dict(_11=7)),
    ("linear", dict(_12=3)), ("linear", dict(_13=9)), ("linear", dict(_5=2 ** 38, _7=2 ** 38, _11=2 ** 38)),
    ("group_norm", dict(_0=0)), ("group_norm", dict(_4=0x3002)), ("group_norm", dict(_11=3)), ("group_norm", dict(_11=0)), ("group_norm", dict(_16=7)), ("group_norm", dict(_17=0)),
    ("group_norm", dict(_18=-1)), ("group_norm", dict(_21=-1.0)), ("group_norm", dict(_21=float("inf"))), ("group_norm", dict(_8=2 ** 40)), ("group_norm", dict(_10=2 ** 21, _16=2 ** 23, _17=2 ** 21)),
    ("gated_delta", dict(_3=0)), ("gated_delta", dict(_5=0x6002)), ("gated_delta", dict(_12=0)), ("gated_delta", dict(_13=3, _12=2)), ("gated_delta", dict(_14=257)), ("gated_delta", dict(_14=0)),
    ("gated_delta", dict(_25=7)), ("gated_delta", dict(_32=63)), ("gated_delta", dict(_33=float("nan"))), ("gated_delta", dict(_35=5)), ("gated_delta", dict(_10=2 ** 40)), ("gated_delta", dict(_16=-4)),
])
def test_entry_points_refuse_before_the_device_is_touched(op, changed):
    L = _lib.load()
    assert getattr(L, "vadc_amd_" + op)(pack(op, **changed), None) == -1
    assert op.encode() in L.vadc_amd_last_error()


def test_entry_points_take_nothing_to_do_and_refuse_a_host_without_a_device():
    L = _lib.load()
    for op, empty in (("linear", dict(_5=0)), ("linear", dict(_7=0, _0=0)), ("group_norm", dict(_9=0, _0=0)), ("gated_delta", dict(_11=0)), ("gated_delta", dict(_10=0, _5=0))):
        assert getattr(L, "vadc_amd_" + op)(pack(op, **empty), None) == 0
    for op in ("linear", "group_norm", "gated_delta"):
        assert getattr(L, "vadc_amd_" + op)(None, None) == -1
    for op in ("group_norm", "gated_delta"):
        assert getattr(L, f"vadc_amd_{op}_workspace")(pack(op)) >= 0
        assert getattr(L, f"vadc_amd_{op}_workspace")(None) == -1
    if not torch.cuda.is_available():
        for op in ("linear", "group_norm", "gated_delta"):
            assert getattr(L, "vadc_amd_" + op)(pack(op), None) == -3
            assert b"no CPU fallback" in L.vadc_amd_last_error()


def test_overlapping_outputs_are_refused():
    x, w = t(4, 8), t(8, 8)

    def spans(*ts):
        return tuple(ops._span(ops._Layout(*ops._layout(a))) for a in ts)

    with pytest.raises(ValueError, match="overlaps x"):
        ops._apart("linear", spans(x, x[1:]), x[1:], (("x", x),))
    with pytest.raises(ValueError, match="overlaps residual"):
        ops._apart("linear", spans(x[:3], x[1:]), x[1:], (("residual", x[:3]),), ("residual",))
    with pytest.raises(ValueError, match="overlaps residual"):               # the same memory in another order
        ops._apart("linear", spans(w, w.T), w.T, (("residual", w),), ("residual",))
    ops._apart("linear", spans(x, x), x, (("residual", x),), ("residual",))
    ops._apart("linear", spans(x[2:], w, x[:2]), x[:2], (("x", x[2:]), ("weight", w)))
    assert issubclass(VadcAmdError, RuntimeError) and C.sizeof(C.c_void_p) == 8


@pytest.mark.parametrize("out, error", [
    (t(4).expand(3, 4), "on top"),
    (torch.zeros(20).as_strided((3, 4), (2, 1)), "on top"),
])
def test_an_output_with_entries_on_top_of_each_other_is_refused(out, error):
    with pytest.raises(ValueError, match=error):
        ops.linear(t(3, 5), t(4, 5), out=out)
    with pytest.raises(ValueError, match=error):
        ops.group_norm(t(3, 4), 2, out=out)


def test_rows_at_one_distance():
    def rows(a):
        return ops._rows("linear", "x", ops._Layout(*ops._layout(a)))

    assert rows(t(6, 5)) == 5 and rows(t(5)) == 5 and rows(t(2, 3, 5)) == 5 and rows(t(6, 9)[:, :5]) == 9
    assert rows(t(2, 1, 3, 9)[..., 2:5]) == 9 and rows(t(1, 4, 9)[:, ::2]) == 18 and rows(t(7, 2, 5)[:, 0]) == 10
    for bad in (t(2, 6, 5)[:, ::2], t(2, 3, 5).transpose(0, 1), t(4, 6, 5)[:, :3]):
        if bad.stride(0) == bad.shape[1] * bad.stride(1):
            continue
        with pytest.raises(ValueError, match="rows"):
            rows(bad)


def test_tensors_share_a_byte_or_not():
    """the overlap of two strided tensors, against the sets of their bytes"""
    import random

    rng, pool = random.Random(5), torch.zeros(4000)
    exact = found = 0
    for _ in range(3000):
        def view():
            dims = rng.randint(1, 3)
            shape = [rng.choice((1, 2, 3, 5)) for _ in range(dims)]
            stride = [rng.choice((0, 1, 2, 3, 4, 6, 8, 20, 24, 40, 120)) for _ in range(dims)]
            return (pool if rng.random() < 0.7 else pool.view(torch.int16)).as_strided(shape, stride, rng.randint(0, 60))

        def held(a):
            at = {(a.data_ptr() - pool.data_ptr())}
            for n, s in zip(a.shape, a.stride()):
                at = {x + i * s * a.element_size() for x in at for i in range(n)}
            return {x + i for x in at for i in range(a.element_size())}

        x, y = view(), view()
        want, got = bool(held(x) & held(y)), ops._shares(x, y)
        assert got or not want                       # an overlap is never missed
        exact += got == want
        found += want
    assert exact > 2950 and 500 < found < 2500, (exact, found)


def test_parts_of_rows_are_apart():
    """an output may lie in the same wide rows as an operand"""
    wide, blocks = t(4, 8), t(2, 5, 4, 6)
    for base, x, y in ((wide, wide[:, :3], wide[:, 3:]), (blocks, blocks[:, :, 1], blocks[:, :, 2:4])):
        assert not ops._shares(x, y) and not ops._shares(y, x)

        def spans(*ts):
            return tuple(ops._span(ops._Layout(*ops._layout(a))) for a in ts)

        ops._apart("linear", spans(x, y), y, (("x", x),))
        with pytest.raises(ValueError, match="overlaps x"):
            ops._apart("linear", spans(base, y), y, (("x", base),))


@pytest.mark.parametrize("name", ("q", "k", "v", "log_decay", "beta", "lengths"))
def test_a_state_that_overlaps_an_input_is_refused(name):
    names = ("q", "k", "v", "log_decay", "beta", "state", "lengths")

    def check(a):
        ts = [a[n] for n in names]
        ops._state_apart(tuple(ops._span(ops._Layout(*ops._layout(x))) for x in ts), *ts)

    a = delta_args(b=2, h=2, dk=4, dv=5, lengths=torch.zeros(2, dtype=torch.int32))
    check(a)
    pool = t(2, 60)                                                  # of each stream 40 values of state, then 20 of something else
    a["state"] = pool.as_strided((2, 2, 4, 5), (60, 20, 5, 1))
    n = min(20, a[name][0].numel())

    def placed(at):
        x = a[name]
        if name == "lengths":
            return pool.view(torch.int32).as_strided((2,), (1,), at)
        return pool.as_strided((2, 1, 1, n) if x.dim() == 4 else (2, 1, n), (60, 20, 20, 1) if x.dim() == 4 else (60, 20, 1), at)

    with pytest.raises(ValueError, match=f"state overlaps {name}"):
        check(dict(a, **{name: placed(39)}))
    check(dict(a, **{name: placed(40)}))                             # between two streams' states


def test_a_tangent_is_refused():
    """forward mode: no result may lose its tangent in silence, under torch.no_grad() either; the same tensors without tangents pass this check"""
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(t(3, 8), t(3, 8))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="linear has no forward-mode derivative"):
                ops._no_tangent("linear", t(3, 8), None, x)
        ops._no_tangent("linear", t(3, 8), forward_ad.unpack_dual(x).primal)
        with forward_ad._set_fwd_grad_enabled(False):
            ops._no_tangent("linear", x)

    def refused(x):
        with pytest.raises(ValueError, match="forward-mode"):
            ops._no_tangent("linear", x)
        return x.sum()

    torch.func.jvp(refused, (t(3),), (t(3),))


def test_a_refusal_does_not_depend_on_what_ran_before():
    """an argument that equals one of a kept plan, but is of a type that is refused"""
    gpu = torch.device("cuda", 0)

    def layout(*shape):
        return (torch.Size(shape), t(*shape).stride(), torch.float32, gpu)

    def norm(groups):
        return ops._plan_norm(layout(3, 8), groups, None, None, 1e-5, "none", None, None, None)

    def linear(first):
        return ops._plan_linear(layout(3, 5), layout(4, 5), None, None, None, "none", first)

    def delta(normalize):
        return ops._plan_delta(layout(2, 3, 1, 4), layout(2, 3, 1, 4), layout(2, 3, 2, 5), layout(2, 3, 2), layout(2, 3, 2), layout(2, 2, 4, 5), None, normalize, None, None)

    for call, good, bad in ((norm, 2, 2.0), (linear, True, 1.0), (delta, False, 0.0)):
        assert call(good) is call(good)
        with pytest.raises(TypeError):
            call(bad)


@pytest.mark.parametrize("what", (None, [[1.0, 2.0]], 3.0, t(3, 5).numpy(), t(3, 5).to_sparse_csr()))
def test_what_is_no_tensor_is_refused(what):
    for call in (lambda: ops.linear(what, t(4, 5)), lambda: ops.linear(t(3, 5), what), lambda: ops.group_norm(what, 1), lambda: ops.gated_delta(**delta_args(log_decay=what)),
                 lambda: ops.gated_delta(**delta_args(state=what))):
        with pytest.raises(TypeError, match="tensor"):
            call()


def test_what_the_library_refuses_is_a_wrong_argument():
    """sizes and strides that only the library looks at: a ValueError with its words, as of every wrong argument"""
    gpu = torch.device("cuda", 0)

    def layout(*shape, dtype=torch.float32):
        stride, n = [], 1
        for d in reversed(shape):
            stride.insert(0, n)
            n *= d
        return (torch.Size(shape), tuple(stride), dtype, gpu)

    with pytest.raises(ValueError, match="group_norm: more than 2\\^20 channels"):
        ops._plan_norm(layout(3, 2 ** 21), 2, None, None, 1e-5, "none", None, None, None)
    steps = 2 ** 27
    with pytest.raises(ValueError, match="gated_delta: more than 2\\^26 steps"):
        ops._plan_delta(layout(1, steps, 1, 4), layout(1, steps, 1, 4), layout(1, steps, 2, 5), layout(1, steps, 2), layout(1, steps, 2), layout(1, 2, 4, 5), None, False, None, None)
    L = _lib.load()
    with pytest.raises(ValueError, match="linear"):
        ops._check(L.vadc_amd_linear(pack("linear", _7=2 ** 25, _11=2 ** 25), None))
    if not torch.cuda.is_available():
        with pytest.raises(VadcAmdError, match="no CPU fallback"):
            ops._check(L.vadc_amd_linear(pack("linear"), None))
