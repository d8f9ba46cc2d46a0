"""Host code of the paged KV cache entry points where the GPU cannot be made to fail: the library's own objects, linked with a
CUDA runtime whose device memory is host memory (fake_cudart.cpp). No GPU is used, and no kernel runs."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

import projectai_b200
from projectai_b200 import build
from projectai_b200.cabi import BackendError, DeviceTimeoutError, NativeBackend, NativeLibrary

HERE = Path(__file__).resolve().parent
OBJECTS = ("context", "paged", "attention_paged", "attention_paged_tc")
TICKETS = 4 * 4096  # bytes of the arrival counters


@pytest.fixture(scope="session")
def fake(tmp_path_factory):
    build.build_cuda()
    out = tmp_path_factory.mktemp("fake") / "libfake.so"
    cuda = Path(build.NVCC).resolve().parents[1]
    subprocess.run([build.CXX, "-shared", "-fPIC", "-std=c++17", "-O1", f"-I{cuda}/include", "-o", str(out), str(HERE / "fake_cudart.cpp"),
                    *[str(build.BUILD / f"{name}.o") for name in OBJECTS], "-Wl,--no-undefined,-Bsymbolic", "-lpthread"], check=True)  # its own runtime, not one that is loaded already
    lib = NativeLibrary(out, "pai_")
    lib.lib.fake_block.argtypes, lib.lib.fake_block.restype = [ctypes.c_size_t], ctypes.c_void_p
    lib.lib.fake_fail_after.argtypes = [ctypes.c_long]
    lib.lib.fake_log.restype = ctypes.c_char_p
    lib.lib.fake_launches.restype = lib.lib.fake_blocks.restype = ctypes.c_long
    return lib


@pytest.fixture()
def be(fake):
    b = NativeBackend(fake)
    yield b
    fake.lib.fake_fail_after(-1)
    b.close()


def device(fake, nbytes, dtype):
    """A block of "device" memory of the newest context, by its size."""
    p = fake.lib.fake_block(nbytes)
    return np.frombuffer((ctypes.c_char * nbytes).from_address(p), dtype=dtype)


def test_an_error_of_the_device_clears_the_arrival_counters(fake, be):
    """A wait that gave up may leave a split item without its last arrival: the counters must not carry that into later
    launches once the error has been read."""
    flag, tickets = device(fake, 64, np.int32), device(fake, TICKETS, np.uint32)
    assert not flag.any() and not tickets.any()  # as created
    for code in (76, 80, 1):
        flag[0], tickets[3], tickets[4095] = code, 2, 1
        with pytest.raises(DeviceTimeoutError):
            be.check_device_error()
        assert flag[0] == 0 and not tickets.any()
    assert be.check_device_error() == 0


def in_use(be):
    n = ctypes.c_int64()
    be._c("memory_stats", ctypes.byref(n), None, None)
    return n.value


def plan_args(be):
    return [be.allocate(s) for s in ((300,), (300,), (300, 2), (700,), (2,))] + [16, 70_000]


def append_args(be):
    q, k, v = be.allocate((700, 8, 64)), be.allocate((700, 2, 64)), be.allocate((700, 2, 64))
    return [q, k, v, be.allocate((9, 64)), be.allocate((9, 64)), be.allocate((700,)), be.allocate((700,)), be.allocate((50, 2, 16, 64)), be.allocate((50, 2, 16, 64))]


def attend_args(be):
    return [be.allocate((700, 8, 64)), be.allocate((50, 2, 16, 64)), be.allocate((50, 2, 16, 64)), be.allocate((3, 9)), be.allocate((4,)),
            be.allocate((3,)), 0.125]


@pytest.mark.parametrize("op,args,allocations", [("paged_plan", plan_args, 5), ("paged_rope_append", append_args, 1), ("sdpa_paged", attend_args, 2)])
def test_a_call_that_runs_out_of_memory_keeps_nothing(fake, be, op, args, allocations):
    args = args(be)
    held, launches = in_use(be), fake.lib.fake_launches()
    for n in range(allocations):  # the allocation that fails
        for scope in (False, True):
            fake.lib.fake_fail_after(0)
            with pytest.raises(MemoryError):  # gives cached blocks back: the next ones are new
                be.allocate((1 << 22,))
            fake.lib.fake_fail_after(n)
            if scope:
                be._c("scope_begin")
            with pytest.raises(MemoryError):
                getattr(be, op)(*args)
            assert in_use(be) == held
            if scope:
                be._c("scope_end")
    assert fake.lib.fake_launches() == launches
    fake.lib.fake_fail_after(-1)
    got = getattr(be, op)(*args)
    assert fake.lib.fake_launches() == launches + 1 and in_use(be) > held
    for t in got if isinstance(got, tuple) else (got,):
        be.release(t)
    assert in_use(be) == held


def test_creating_a_context_waits_for_nothing_but_its_own_stream(fake):
    """Whatever else the device does, a graph capture of another context included."""
    fake.lib.fake_log_clear()
    b = NativeBackend(fake)
    assert fake.lib.fake_log() == b""
    assert not device(fake, 64, np.int32).any() and not device(fake, TICKETS, np.uint32).any()
    b.close()


def test_a_context_that_runs_out_of_memory_keeps_nothing(fake):
    held = fake.lib.fake_blocks()
    for n in range(2):
        fake.lib.fake_fail_after(n)
        with pytest.raises(BackendError):
            NativeBackend(fake)
        assert fake.lib.fake_blocks() == held
    fake.lib.fake_fail_after(-1)
