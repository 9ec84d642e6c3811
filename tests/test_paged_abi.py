"""The paged cache's host side without a GPU: sizes, structs and refusals, and
the plain form's own layout."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch  # noqa: F401  before the library, which then shares torch's HIP runtime

from rustyllm_amd import hip
from tests import paged_ref as R


@pytest.mark.parametrize("hd,vd,g", [(8, 8, 2), (64, 64, 2), (72, 64, 4), (128, 128, 4), (64, 136, 8), (256, 256, 8)])
def test_pool_bytes(hd, vd, g):
    assert hip.paged_kv_bytes(7, 48, 3, hd, vd) == 7 * 48 * 3 * 18 * g == R.Pool(7, 48, 3, hd, vd).k.size


@pytest.mark.parametrize("args", [(0, 16, 1, 64), (1, 0, 1, 64), (1, 24, 1, 64), (1, 65552, 1, 64), (1, 16, 0, 64),
                                  (1, 16, 1, 0), (1, 16, 1, 60), (1, 16, 1, 264), (1, 16, 1, 64, 4),
                                  (1 << 31, 16, 1, 64)])
def test_pool_sizes_refused(args):
    assert hip.paged_kv_bytes(*args) == 0


def test_large_pool_bytes_do_not_wrap():
    assert hip.paged_kv_bytes((1 << 31) - 1, 65536, 4096, 256) == 0
    assert hip.paged_kv_bytes(1 << 20, 64, 8, 128) == (1 << 20) * 64 * 8 * 72


def test_struct_layouts():
    """Offsets of the C structs (include/rusty_hip.h) on a 64-bit host."""
    assert C.sizeof(hip._PagedKv) == 56 and hip._PagedKv.n_pages.offset == 32
    assert C.sizeof(hip._PagedBatch) == 64 and hip._PagedBatch.n_seqs.offset == 48
    assert hip._PagedAppend.cos_t.offset == 112 and C.sizeof(hip._PagedAppend) == 152
    assert hip._PagedRead.k.offset == 8 and C.sizeof(hip._PagedRead) == 56
    assert hip._PagedAttention.scale.offset == 80 and C.sizeof(hip._PagedAttention) == 104


@pytest.mark.parametrize("packed,fields", [("_PAGED_APPEND", "_PagedAppend"), ("_PAGED_READ", "_PagedRead"),
                                           ("_PAGED_ATTENTION", "_PagedAttention")])
def test_packed_rows_are_the_struct(packed, fields):
    """pack() writes every field where the struct has it."""
    fmt, struct = getattr(hip, packed), getattr(hip, fields)
    values = [0.5 if t is C.c_float else 3 + i for i, (_, t) in enumerate(struct._fields_)]
    data = fmt.pack(*values).ljust(C.sizeof(struct), b"\0")
    got = struct.from_buffer_copy(data)
    assert [getattr(got, name) for name, _ in struct._fields_] == values


class _Call:
    """Structs that would be taken, over addresses that are never followed: every
    refusal comes before any device is looked for."""

    def __init__(self):
        size = hip.paged_kv_bytes(9, 32, 2, 64)
        self.kv = hip._PagedKv(4096, 8192, size, size, 9, 32, 2, 64, 64)
        self.batch = hip._PagedBatch(4096, 4096, 4096, 2 * 5 * 4, 8, 12, 2, 5, 2, 100)
        row = 2 * 64 * 4
        self.append = hip._PagedAppend(0, 3, 4, 4096, 4096, 4096, 4096, 6 * row, 3 * row, 3 * row, 6 * row, 256, 128, 128,
                                       256, 4096, 4096, 100 * 32 * 4, 100, 64, 0)
        self.read = hip._PagedRead(0, 3, 4096, 4096, 3 * row, 3 * row, 128, 128)
        self.attn = hip._PagedAttention(0, 3, 4, 4096, 4096, 6 * row, 6 * row, 256, 256, None, 0, 0.125, 0, 4096, 1 << 30)

    def all(self):
        L, r = hip.lib, C.addressof
        return [L.rusty_hip_paged_append(r(self.kv), r(self.batch), r(self.append), None),
                L.rusty_hip_paged_read(r(self.kv), r(self.batch), r(self.read), None),
                L.rusty_hip_paged_attention(r(self.kv), r(self.batch), r(self.attn), None)]


@pytest.mark.parametrize("struct,field,value", [
    ("kv", "k_pages", None), ("kv", "v_pages", None), ("kv", "k_pages", 4097), ("kv", "k_len", 100), ("kv", "v_len", 0),
    ("kv", "n_pages", 0), ("kv", "page_size", 24), ("kv", "n_kv_heads", 0), ("kv", "head_dim", 260),
    ("kv", "value_dim", 12), ("batch", "page_table", None), ("batch", "kv_lens", None), ("batch", "q_starts", None),
    ("batch", "page_table_len", 39), ("batch", "kv_lens_len", 7), ("batch", "q_starts_len", 8), ("batch", "n_seqs", 0),
    ("batch", "table_stride", 0), ("batch", "max_q_len", 0), ("batch", "kv_lens", 4098),
    ("batch", "n_seqs", 1 << 25), ("batch", "table_stride", 1 << 25),
])
def test_refused_by_every_call(struct, field, value):
    c = _Call()
    setattr(getattr(c, struct), field, value)
    assert c.all() == [0, 0, 0]


@pytest.mark.parametrize("struct,at,field,value", [
    ("append", 0, "n_rows", 0), ("append", 0, "n_rows", 1 << 25), ("append", 0, "n_rows", 4), ("read", 1, "n_rows", 0),
    ("read", 1, "n_rows", 4), ("attn", 2, "n_rows", 0), ("attn", 2, "n_rows", 4),
    ("append", 0, "dtype", 2), ("append", 0, "k", None), ("append", 0, "v", None), ("append", 0, "q_out", None),
    ("append", 0, "n_heads", 3), ("append", 0, "n_heads", 0), ("append", 0, "q_len", 3071), ("append", 0, "k_len", 10),
    ("append", 0, "k_stride", 126), ("append", 0, "k_stride", 64), ("append", 0, "v_stride", -128),
    ("append", 0, "k", 4100), ("append", 0, "cos_t", None), ("append", 0, "sin_t", 4104), ("append", 0, "table_len", 99),
    ("append", 0, "max_pos", 0), ("append", 0, "rot_dim", 24), ("append", 0, "rot_dim", 80), ("read", 1, "dtype", 9),
    ("read", 1, "k_len", 8), ("read", 1, "v_stride", 2), ("attn", 2, "dtype", 2), ("attn", 2, "q", None),
    ("attn", 2, "out", None), ("attn", 2, "n_heads", 5), ("attn", 2, "q_len", 16), ("attn", 2, "out_stride", 255),
    ("attn", 2, "out", 4104), ("attn", 2, "window", 1 << 31), ("attn", 2, "scale", float("nan")),
    ("attn", 2, "q_stride", 1 << 50),
])
def test_refused_rows(struct, at, field, value):
    c = _Call()
    setattr(getattr(c, struct), field, value)
    assert c.all()[at] == 0


def test_null_structs_are_refused():
    L, c = hip.lib, _Call()
    r = C.addressof
    for f, rows in ((L.rusty_hip_paged_append, c.append), (L.rusty_hip_paged_read, c.read),
                    (L.rusty_hip_paged_attention, c.attn)):
        assert f(None, r(c.batch), r(rows), None) == 0
        assert f(r(c.kv), None, r(rows), None) == 0
        assert f(r(c.kv), r(c.batch), None, None) == 0
    c.read.k = c.read.v = None
    assert c.all()[1] == 0


def test_without_a_gpu_nothing_is_handled():
    from tests.conftest import gpu_present
    if gpu_present():
        pytest.skip("GPU present")
    assert _Call().all() == [0, 0, 0]


def test_workspace_grows_with_the_split():
    c = _Call()
    f = lambda: hip.lib.rusty_hip_paged_attention_workspace(C.addressof(c.kv), C.addressof(c.batch), 3, 4)  # noqa: E731
    c.batch.max_kv_len = 16
    small = f()
    c.batch.max_kv_len = 100000
    assert f() > small
    c.batch.n_seqs = 0
    assert f() == 0


def test_plain_form_round_trip():
    """What the host pool stores it loads, and quantization is off by at most half a
    step, a whole one at the end of the range without a code of its own."""
    rng = np.random.default_rng(0)
    p = R.Pool(3, 16, 2, 80, 96)
    for off in (0, 3, 15):
        for which, dim in (("k", 80), ("v", 96)):
            x = rng.standard_normal((2, dim)).astype(np.float32)
            p.store(which, 2, off, x)
            got = p.load(which, 2, off)
            for g in range(0, dim, 32):
                step = np.abs(x[:, g:g + 32]).max(1) / 8 * (1 + 2.0 ** -10)
                assert (np.abs(got - x)[:, g:g + 32] <= step[:, None] * 1.01).all()
    assert np.isnan(p.load("k", 1, 4)).all()


def test_attention_of_the_plain_form_is_softmax():
    rng = np.random.default_rng(1)
    p = R.Pool(4, 16, 1, 8)
    table = np.array([[2, 0, 3]], np.int32)
    for t in range(35):
        p.store("k", table[0, t // 16], t % 16, rng.standard_normal((1, 8)).astype(np.float32))
        p.store("v", table[0, t // 16], t % 16, rng.standard_normal((1, 8)).astype(np.float32))
    k = np.stack([p.load("k", table[0, t // 16], t % 16)[0] for t in range(35)])
    v = np.stack([p.load("v", table[0, t // 16], t % 16)[0] for t in range(35)])
    q = rng.standard_normal((2, 2, 8)).astype(np.float32)
    out, _, _ = R.attention(p, table, [35], [0, 2], q, 0.3)
    for r in range(2):
        w = np.exp(0.3 * k[:34 + r] @ q[r].T.astype(np.float64))
        assert np.allclose(out[r], (w / w.sum(0)).T @ v[:34 + r], rtol=1e-12)


@pytest.mark.parametrize("first,second,refused", [("torch", "rustyllm_amd.hip", False),
                                                  ("rustyllm_amd.hip", "torch", True)])
def test_two_hip_runtimes_are_refused(first, second, refused):
    """torch brings a HIP runtime of its own: loaded behind the library there are two
    in the process, and a stream or tensor of one means nothing to the other."""
    code = (f"import {first}, {second}\nimport torch\nfrom rustyllm_amd import hip\n"
            "t = torch.zeros(hip.paged_kv_bytes(1, 16, 1, 64), dtype=torch.uint8)\n"
            "try:\n    hip.PagedKv(t, t, 1, 16, 1, 64)\n"
            "except Exception as e:\n    print(type(e).__name__)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    # a CPU tensor is a ValueError, once the runtimes are found to be one
    assert run.stdout.strip() == ("RuntimeError" if refused else "ValueError"), run.stderr
