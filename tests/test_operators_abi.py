"""The operators' C entry points refuse wrong arguments before they look for a device, and a machine without one."""
import ctypes as C
import subprocess
import sys

import pytest

P, U, W, I, F = C.c_void_p, C.c_uint64, C.c_uint32, C.c_int, C.c_float


@pytest.fixture(scope="module")
def lib(cp):
    lib = cp.load_library()
    for name in ("embedding_grad", "int8_matmul", "distill"):
        getattr(lib, "cphnsw_b200_%s_workspace" % name).restype = U
    return lib


def p(v):
    return P(v)


A = 1 << 20  # an address that nothing reads: every call below fails before a launch


def lookup(table=A, type=0, rows=10, dim=8, stride=8, ids=A, id_bytes=4, n=3, out=A, out_stride=8):
    return (p(table), I(type), U(rows), U(dim), U(stride), p(ids), W(id_bytes), U(n), F(1.0), p(out), U(out_stride), p(0))


def grad(ids=A, id_bytes=4, n=3, g=A, type=0, stride=8, out=A, out_type=0, rows=10, dim=8, out_stride=8, ws=0, ws_bytes=0):
    return (p(ids), W(id_bytes), U(n), p(g), I(type), U(stride), F(1.0), p(out), I(out_type), U(rows), U(dim), U(out_stride), I(0), p(ws), U(ws_bytes), p(0))


def quantize(x=A, type=0, n=3, dim=8, stride=8, q=A, q_stride=16, scale=A):
    return (p(x), I(type), U(n), U(dim), U(stride), p(q), U(q_stride), p(scale), p(0))


def matmul(a=A, a_stride=16, sa=A, m=3, b=A, b_stride=16, sb=A, n=5, k=16, out=A, type=2, out_stride=5, ws=0, ws_bytes=0):
    return (p(a), U(a_stride), p(sa), U(m), p(b), U(b_stride), p(sb), U(n), U(k), p(out), I(type), U(out_stride), p(ws), U(ws_bytes), p(0))


def loss(z=A, type=0, n=3, rows=10, stride=10, ids=A, id_bytes=4, teacher=A, top=4, T=1.0, out=A):
    return (p(z), I(type), U(n), U(rows), U(stride), p(ids), W(id_bytes), U(top), p(teacher), U(top), U(top), F(T), p(out), p(0))


def step(z=A, type=0, n=3, rows=10, stride=10, ids=A, id_bytes=4, teacher=A, top=4, T=1.0, weight=0, out=A, g=A, g_stride=10, ws=A, ws_bytes=1 << 20):
    return (p(z), I(type), U(n), U(rows), U(stride), p(ids), W(id_bytes), U(top), p(teacher), U(top), U(top), F(T), p(weight), p(out), p(g), U(g_stride),
            p(ws), U(ws_bytes), p(0))


CALLS = [
    ("embedding_lookup_dev", lookup, [dict(table=0), dict(ids=0), dict(out=0), dict(type=3), dict(rows=0), dict(rows=1 << 31), dict(dim=0), dict(id_bytes=2),
                                      dict(out_stride=7), dict(table=A + 2), dict(ids=A + 2), dict(ids=A + 4, id_bytes=8)]),
    ("embedding_grad_dev", grad, [dict(ids=0), dict(g=0), dict(out=0), dict(type=1, out_type=2), dict(type=0, out_type=1), dict(rows=0), dict(dim=0),
                                  dict(n=1 << 31), dict(out_stride=7), dict(n=5000), dict(n=5000, ws=A + 16, ws_bytes=1 << 30), dict(g=A + 2)]),
    ("quantize_rows_dev", quantize, [dict(x=0), dict(q=0), dict(scale=0), dict(type=-1), dict(dim=0), dict(q_stride=7), dict(scale=A + 2), dict(x=A + 1)]),
    ("int8_matmul_dev", matmul, [dict(a=0), dict(b=0), dict(sa=0), dict(sb=0), dict(out=0), dict(k=0), dict(k=131_072), dict(m=1 << 31), dict(n=1 << 31),
                                 dict(out_stride=4), dict(type=7), dict(a=A + 1), dict(b_stride=17), dict(a_stride=20, ws=A + 8, ws_bytes=1 << 20)]),
    ("distill_loss_dev", loss, [dict(z=0), dict(ids=0), dict(teacher=0), dict(out=0), dict(type=5), dict(rows=0), dict(top=1025), dict(T=0.0), dict(T=-1.0),
                                dict(T=float("nan")), dict(T=float("inf")), dict(id_bytes=1), dict(z=A + 2), dict(n=1 << 31)]),
    ("distill_loss_and_grad_dev", step, [dict(g=0), dict(g_stride=9), dict(ws=0, ws_bytes=0), dict(ws=A + 8), dict(ws_bytes=10), dict(weight=A + 2),
                                         dict(top=1025), dict(T=0.0), dict(rows=1 << 31)]),
]


@pytest.mark.parametrize("name,build,wrong", CALLS, ids=[c[0] for c in CALLS])
def test_wrong_arguments(cp, lib, name, build, wrong):
    fn = getattr(lib, "cphnsw_b200_" + name)
    for kwargs in wrong:
        assert fn(*build(**kwargs)) == cp.E_INVALID, kwargs
        assert name[:-4] in lib.cphnsw_b200_last_error().decode() or "distill" in name
    # nothing to do is no error, device or not
    empty = dict(m=0, out_stride=5) if name == "int8_matmul_dev" else dict(n=0)
    if name != "embedding_grad_dev":  # (a gradient of no places is written as zeros)
        assert fn(*build(**empty)) == 0


def test_without_a_device(cp, lib):
    if cp.device_count() > 0:
        pytest.skip("a GPU is present")
    for name, build, _ in CALLS:
        assert getattr(lib, "cphnsw_b200_" + name)(*build()) == cp.E_CUDA
        assert "no CPU path" in lib.cphnsw_b200_last_error().decode()
    assert lib.cphnsw_b200_operator_status() == cp.E_CUDA


def test_workspaces(lib):
    assert lib.cphnsw_b200_embedding_grad_workspace(U(100), U(1000), U(64)) == 0
    small, large = (lib.cphnsw_b200_embedding_grad_workspace(U(n), U(1000), U(64)) for n in (5000, 50_000))
    assert 0 < small < large
    assert lib.cphnsw_b200_int8_matmul_workspace(p(A), U(64), U(8), p(A), U(64), U(8), U(64)) == 0
    # rows of 100 bytes are copied to rows of 112, 256 bytes at a time
    assert lib.cphnsw_b200_int8_matmul_workspace(p(A), U(100), U(8), p(A), U(112), U(8), U(100)) == 1024
    assert lib.cphnsw_b200_distill_workspace(U(10), U(64)) >= 10 * 64 * 12


def test_workspaces_of_refused_sizes(cp):
    """Sizes that the calls refuse are answered too, and at once (a process of its own: one that does not answer is ended)."""
    code = """
import ctypes as C, sys
fn = C.CDLL(sys.argv[1]).cphnsw_b200_embedding_grad_workspace
fn.restype = C.c_uint64
for n, rows, dim in [(5000, 2**64 - 1, 8), (5000, 2**63, 8), (5000, 2**31, 8), (2**31, 100, 8), (2**64 - 1, 100, 8), (5000, 100, 2**20)]:
    assert fn(C.c_uint64(n), C.c_uint64(rows), C.c_uint64(dim)) == 0, (n, rows, dim)
assert fn(C.c_uint64(5000), C.c_uint64(2**31 - 1), C.c_uint64(8)) > 2**31 * 4
"""
    done = subprocess.run([sys.executable, "-c", code, cp.LIB_PATH], timeout=60, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
