"""The serving operators on the host: refusals of every entry point
(tests/cpp/test_serving_args.cpp, with a context of a device that is not there),
where a batch's tokens stand whatever its arrays hold (tests/cpp/test_kvindex.cpp),
and the tables of scaled frequencies against their closed forms."""
import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import mimir_hip as M

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.dirname(M.LIB_PATH)
ROCM = "/opt/rocm"


def build_and_run(tmp_path, name, *flags):
    exe = tmp_path / name
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-o", str(exe), os.path.join(HERE, "cpp", name + ".cpp"), *flags],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert " 0 failures" in r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_positions_and_pages(tmp_path):
    build_and_run(tmp_path, "test_kvindex", "-Werror")


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(ROCM), reason="g++ or ROCm not available")
def test_refusals(tmp_path):
    build_and_run(tmp_path, "test_serving_args", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include", f"-L{LIB}", "-lmimir_hip",
                  f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{LIB}", f"-Wl,-rpath,{ROCM}/lib")


def test_null_context_is_einval():
    lib = M.load()
    cache, batch, rope = M._lib.KVCache_C(), M._lib.KVBatch_C(), M._lib.Rope_C()
    assert lib.mimir_kv_append(None, cache, batch, None, None, 0, rope, None, 0, None, 0, 0) == M.EINVAL
    assert lib.mimir_kv_read(None, cache, batch, None, None, 0) == M.EINVAL
    assert lib.mimir_attention_paged_fwd(None, cache, batch, None, 0, None, 0, 1, 1.0, 1) == M.EINVAL
    assert lib.mimir_rope_rows_fwd(None, None, 0, None, 0, 0, None, 0, None, 0, 0, 0, 8, None, rope) == M.EINVAL
    assert lib.mimir_rope_rows_bwd(None, None, 0, None, 0, 0, None, 0, None, 0, 0, 0, 8, None, rope, 0) == M.EINVAL


class Room:
    """A context's allocations without a GPU: `most` buffers, then MimirError."""

    def __init__(self, most):
        self.lib, self.most, self.held = M.load(), most, {}

    def empty(self, shape, dtype=np.float32):
        if len(self.held) == self.most:
            raise M.MimirError(M.ENOMEM, "no room")
        a = M.DeviceArray(self, 16 * (len(self.held) + 1), shape, dtype)
        self.held[a.ptr] = a
        return a

    def free(self, a):
        del self.held[a.ptr]


@pytest.mark.parametrize("dtype,buffers", [("f32", 2), ("bf16", 2), ("i8", 4)])
def test_a_cache_without_room_keeps_nothing(dtype, buffers):
    for most in range(buffers):
        room = Room(most)
        with pytest.raises(M.MimirError):
            M.KVCache(room, dtype, 3, 16, 2, 20)
        assert not room.held
    room = Room(buffers)
    cache = M.KVCache(room, dtype, 3, 16, 2, 20)
    assert len(room.held) == buffers and cache.c.k == cache.k.ptr and cache.c.v_scale == (cache.v_scale.ptr if buffers == 4 else None)
    cache.close()
    cache.close()
    assert not room.held


@pytest.mark.parametrize("dtype", ["f32", "bf16", "i8"])
def test_a_closed_cache_is_refused(dtype):
    """Its buffers are gone: no address of theirs is left for a call to take."""
    room = Room(4)
    cache = M.KVCache(room, dtype, 3, 16, 2, 20)
    cache.close()
    assert cache.c.k is None and cache.c.v is None and cache.c.k_scale is None and cache.c.v_scale is None
    given = M.KVCache(room, dtype, 3, 16, 2, 20, 64, 128, 192, 256)
    given.close()  # the program's own buffers stay its own
    assert given.c.k == 64 and given.c.v == 128


def frequencies(rot, theta, kind, factor, original_len, low, high):
    if kind == "base":
        theta = theta * factor ** (rot / (rot - 2))
    f = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind == "by_parts":
        g = [min(1.0, max(0.0, (original_len * x / (2 * math.pi) - low) / (high - low))) for x in f]
        f = [(1 - a) * x / factor + a * x for x, a in zip(f, g)]
    return f


@pytest.mark.parametrize("kind", ["none", "linear", "base", "by_parts"])
@pytest.mark.parametrize("rot,theta,first", [(8, 1e4, 0), (64, 5e5, 120000), (128, 1e4, 3)])
def test_scaled_tables(kind, rot, theta, first):
    """A table value is off by half a step of fp32 and by the angle's own error: the
    frequency is right to a few steps of a double, 1e-15, times a position of 2^17."""
    args = dict(factor=8.0, original_len=4096.0, low=1.0, high=32.0)
    c, s = M.rope_table_scaled(5, rot, theta, kind=kind, magnitude=1.2, first=first, **args)
    f = frequencies(rot, theta, kind, *args.values())
    for p in range(5):
        for i in range(rot // 2):
            a = (first + p) * f[i]
            for got, want in ((c[p, i], 1.2 * math.cos(a)), (s[p, i], 1.2 * math.sin(a))):
                assert abs(float(got) - want) <= 2.0 ** -24 * 1.2 + 1.2 * 2.0 ** 17 * 4e-15


@pytest.mark.parametrize("args", [
    dict(kind="linear", factor=1e-320),                    # f / factor
    dict(kind="linear", factor=1e-306, first=1 << 40),     # the angle
    dict(kind="base", factor=1e-300, rot_dim=4),           # theta * factor^2
    dict(kind="by_parts", factor=1e-320, original_len=8, low=1, high=2),
    dict(theta=1e-320, rot_dim=64),
    dict(magnitude=1e39),
    dict(first=(1 << 63) - 2),                             # the last position
])
def test_tables_that_would_not_be_finite_are_refused(args):
    lib = M.load()
    how = dict(rot_dim=8, theta=1e4, kind="none", factor=1.0, original_len=1.0, low=1.0, high=32.0, magnitude=1.0, first=0) | args
    c = np.full((5, how["rot_dim"] // 2), 7.0, np.float32)
    z = M._lib.RopeScaling_C(M._lib.ROPE_SCALINGS.index(how["kind"]), how["factor"], how["original_len"], how["low"], how["high"],
                             how["magnitude"])
    at = c.ctypes.data_as(ctypes.c_void_p)
    assert lib.mimir_rope_table_scaled(how["first"], 5, how["rot_dim"], how["theta"], ctypes.byref(z), at, at) == M.EINVAL
    assert (c == 7).all()


def test_unscaled_table_is_rope_table():
    for a, b in zip(M.rope_table_scaled(40, 64, 1e4), M.rope_table(40, 64, 1e4)):
        np.testing.assert_array_equal(a, b)


def test_by_parts_keeps_fast_pairs_and_stretches_slow_ones():
    _, s = M.rope_table_scaled(2, 64, 1e4, kind="by_parts", factor=4.0, original_len=4096, low=1, high=32)
    _, plain = M.rope_table(2, 64, 1e4)
    _, linear = M.rope_table_scaled(2, 64, 1e4, kind="linear", factor=4.0)
    assert s[1, 0] == plain[1, 0] and s[1, -1] == linear[1, -1]
