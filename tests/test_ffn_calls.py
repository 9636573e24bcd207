"""How the feed-forward entry points are called: memory that calls leave, what the wrapper refuses, the binding's
build."""
import os

import numpy as np
import pytest

from tests.test_ffn import SIZES, operands


@pytest.fixture(scope="module")
def lib():
    from exo_b200 import build

    build.build()
    import exo_b200

    return exo_b200.library()


# ------------------------------------------------------------------ memory of operand copies
def test_trim_without_a_device_is_an_error(lib):
    import torch

    import exo_b200

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(exo_b200.ExoB200Error) as e:
        lib.trim()
    assert e.value.code in (exo_b200.ERR_CUDA, exo_b200.ERR_UNSUPPORTED)


@pytest.mark.gpu
def test_trim_gives_the_copies_memory_back(lib):
    """Weights of an odd pitch are copied into the context's pool, which keeps the memory for the next call until it is
    trimmed; what calls in a context of its own leave is that context's.  Results do not depend on it."""
    import torch

    import exo_b200

    M, F, K = 64, 16384, 4095  # 2 * 134 MB of copies
    x, wg, wu = (torch.randn(s, device="cuda").bfloat16() * 0.02 for s in ((M, K), (F, K), (F, K)))
    h, again = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ctx = exo_b200.Context()

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]

    for c in (None, ctx):
        lib.trim(c)
        before = free()
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, h, None, None)
        kept = before - free()
        assert kept >= 2 * F * K * 2
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, again, None, None)
        assert before - free() == kept and torch.equal(h, again)
        lib.trim(c)
        # (a first call of a kernel may have loaded its code: some MB at most)
        assert before - free() < 64 << 20
        again.zero_()
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, again, None, None)
        torch.cuda.synchronize()
        assert torch.equal(h, again)
        lib.trim(c)
    # trimmed while work is enqueued: its copies stay
    for _ in range(20):
        lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, again, None, None)
        lib.trim()
    torch.cuda.synchronize()
    assert torch.equal(h, again)
    lib.trim()


@pytest.mark.gpu
def test_graphs_with_copies_run_beside_one_another(lib):
    """Two graphs whose calls copy operands, replayed on two streams at once, trimmed in between, while eager calls of
    another size go through a third stream: each has memory of its own."""
    import torch

    M, F, K = 200, 1333, 517
    wg, wu = (torch.randn(F, K, device="cuda").bfloat16() * 0.05 for _ in range(2))
    x = [torch.randn(M, K, device="cuda").bfloat16() for _ in range(2)]
    want, got = ([torch.zeros(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2))
    big = [torch.randn(s, device="cuda").bfloat16() for s in ((300, 519), (2000, 519), (2000, 519))]
    other, other_want = (torch.zeros(300, 2000, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for xi, w in zip(x, want):
        lib.gated_bf16_exo(None, 1, M, F, K, xi, wg, wu, w, None, None)
    lib.gated_bf16_exo(None, 1, 300, 2000, 519, *big, other_want, None, None)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for xi, g in zip(x, got):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lib.gated_bf16_exo(None, 1, M, F, K, xi, wg, wu, g, None, None)
        graphs.append(graph)
    for turn in range(10):
        for g in (*got, other):
            g.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                lib.gated_bf16_exo(None, 1, 300, 2000, 519, *big, other, None, None)
        if turn % 3 == 1:
            lib.trim()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(other, other_want)
        if turn % 3 == 2:
            lib.trim()


@pytest.mark.gpu
def test_a_thread_may_capture_while_another_calls(lib):
    """One thread captures calls with copies while another one's calls grow the context's pool."""
    import threading

    import torch

    M, F, K = 64, 333, 257
    x, wg, wu = (torch.randn(s, device="cuda").bfloat16() for s in ((M, K), (F, K), (F, K)))
    h, want = (torch.zeros(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, want, None, None)
    big = [torch.randn(s, device="cuda").bfloat16() for s in ((64, 1001), (9001, 1001), (9001, 1001))]
    wide, wide_want = (torch.zeros(64, 9001, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lib.gated_bf16_exo(None, 0, 64, 9001, 1001, *big, wide_want, None, None)
    torch.cuda.synchronize()
    lib.trim()
    captured, called, failed = threading.Event(), threading.Event(), []

    def work():
        try:
            captured.wait(60)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    lib.gated_bf16_exo(None, 0, 64, 9001, 1001, *big, wide, None, None)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
        finally:
            called.set()

    thread = threading.Thread(target=work)
    thread.start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, h, None, None)
        captured.set()
        assert called.wait(60)
        lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, h, None, None)
    thread.join()
    graph.replay()
    torch.cuda.synchronize()
    assert not failed, failed
    assert torch.equal(h, want) and torch.equal(wide, wide_want)


# ------------------------------------------------------------------ build of the binding's fast path
@pytest.fixture
def call_at(tmp_path, monkeypatch):
    """build.build_call into a directory of its own."""
    import sysconfig

    from exo_b200 import build

    monkeypatch.setattr(build, "CALL", str(tmp_path / os.path.basename(build.CALL)))
    assert os.path.basename(build.CALL) == "_call" + sysconfig.get_config_var("EXT_SUFFIX")
    return tmp_path, build


def test_the_fast_path_is_built_for_this_interpreter(call_at):
    import importlib.util

    path, build = call_at
    (path / "_call.so").write_bytes(b"of some interpreter")
    (path / "_call.cpython-30-x86_64-linux-gnu.so").write_bytes(b"of another, older than the source")
    os.utime(path / "_call.cpython-30-x86_64-linux-gnu.so", (1, 1))
    (path / "_call.cpython-31-x86_64-linux-gnu.so").write_bytes(b"of another")
    made = build.build_call()
    assert sorted(os.listdir(path)) == sorted(["_call.cpython-31-x86_64-linux-gnu.so", os.path.basename(made)])
    spec = importlib.util.spec_from_file_location("_call", made)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert callable(module.call)
    before = os.stat(made).st_mtime_ns
    assert build.build_call() == made and os.stat(made).st_mtime_ns == before


@pytest.mark.parametrize("compiler", ["/nowhere/c++", "false"])
def test_no_compiler_is_no_error_and_leaves_no_old_module(call_at, monkeypatch, capsys, compiler):
    path, build = call_at
    monkeypatch.setenv("CXX", compiler)
    with open(build.CALL, "wb") as f:
        f.write(b"of an older source")
    os.utime(build.CALL, (1, 1))
    assert build.build_call() is None
    assert os.listdir(path) == [] and "fast path is not built" in capsys.readouterr().err
    with open(build.CALL, "wb") as f:
        f.write(b"of this source")
    assert build.build_call(force=True) is None  # one that is up to date stays
    assert os.listdir(path) == [os.path.basename(build.CALL)]


def test_no_headers_is_no_error_and_leaves_no_old_module(call_at, monkeypatch):
    import sysconfig

    path, build = call_at
    with open(build.CALL, "wb") as f:
        f.write(b"of an older source")
    os.utime(build.CALL, (1, 1))
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(path / "none")})
    assert build.build_call() is None
    assert os.listdir(path) == []


# ------------------------------------------------------------------ what the wrapper refuses
def test_a_torch_without_uint16_will_do(lib, monkeypatch):
    """torch before 2.3 has no uint16, and a module that is still being imported has nothing yet."""
    import sys
    import types

    import torch

    import exo_b200
    from exo_b200 import api

    old = types.ModuleType("torch")
    for name in ("Tensor", "nn", "bfloat16", "int16", "int8", "float32"):
        setattr(old, name, getattr(torch, name))
    old._C = types.SimpleNamespace()
    for module, torch_known in ((old, True), (types.ModuleType("torch"), False)):
        monkeypatch.setitem(sys.modules, "torch", module)
        proc = api.CheckedProc(lib.dll, "gated_bf16_exo")
        ops = operands("gated_bf16_exo", SIZES["gated_bf16_exo"])
        with pytest.raises(ValueError, match="has 4 elements"):
            proc(None, 0, 3, 4, 5, np.ones(4, np.uint16), *ops[1:])
        with pytest.raises(exo_b200.ExoB200Error):  # arrays pass the wrapper
            proc(None, 0, 3, 4, 5, None, *ops[1:])
        if torch_known:
            tensors = [torch.ones(o.shape, dtype=torch.bfloat16) for o in ops]
            with pytest.raises(exo_b200.ExoB200Error):
                proc(None, 0, 3, 4, 5, None, *tensors[1:])


def shapes_of(name, rows, width):
    """Shapes of rows * width elements, and whether their last dimension is the row."""
    return [((rows * width,), True), ((rows, width), True), ((1, rows, width), True), ((width, rows), False),
            ((1, rows * width), False), ((rows * width, 1), False)]


def check_shapes(call, name, make):
    """Every operand of `name` in every shape: the right ones pass the wrapper (and are refused behind it, for an operand
    that is missing), the others do not."""
    import exo_b200
    from exo_b200 import _lib

    sizes = SIZES[name]
    specs = _lib.SIGNATURES[name][1]
    ops = [make([sizes[d] for d in dims], kind) for kind, _, dims in specs]
    required = [i for i, (_, optional, _) in enumerate(specs) if not optional]
    for i, (kind, _, dims) in enumerate(specs):
        missing = next(k for k in reversed(required) if k != i)
        shapes = shapes_of(name, *(sizes[d] for d in dims)) if len(dims) == 2 else [((sizes[dims[0]], 1), True)]
        for shape, right in shapes:
            args = [None if k == missing else make(shape, kind) if k == i else o for k, o in enumerate(ops)]
            if right:
                with pytest.raises(exo_b200.ExoB200Error) as e:
                    call(None, *sizes, *args)
                assert e.value.code == exo_b200.ERR_INVALID_ARGUMENT
            else:
                with pytest.raises(ValueError, match=f"operand {i + 1} has rows of {shape[-1]} elements, not"):
                    call(None, *sizes, *args)


TYPES = {"bf16": ("uint16", "bfloat16"), "i8": ("int8", "int8"), "f32": ("float32", "float32")}


@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_transposed_operands(lib, name):
    """[K, F] where [F, K] is meant has the right count and the wrong rows."""
    import torch

    check_shapes(getattr(lib, name), name, lambda shape, kind: np.ones(shape, TYPES[kind][0]))
    check_shapes(getattr(lib, name), name, lambda shape, kind: torch.ones(shape, dtype=getattr(torch, TYPES[kind][1])))


@pytest.mark.gpu
@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_transposed_device_operands(lib, name):
    import torch

    check_shapes(getattr(lib, name), name,
                 lambda shape, kind: torch.ones(shape, dtype=getattr(torch, TYPES[kind][1]), device="cuda"))
    assert getattr(lib, name)._fast is not None


@pytest.mark.gpu
def test_the_fast_path_takes_every_right_shape(lib):
    import torch

    from exo_b200 import api

    x, s = torch.randn(6, 8, device="cuda"), torch.zeros(6, device="cuda")
    q = torch.zeros(6, 8, dtype=torch.int8, device="cuda")
    lib.quantize_rows_f32_exo(None, 6, 8, x, q, s)
    for shape in ((48,), (6, 8), (2, 3, 8), (1, 6, 8)):
        again, t = torch.zeros_like(q).view(shape), torch.zeros(3, 2, device="cuda")
        assert api._call.call(lib.quantize_rows_f32_exo._fast, (None, 6, 8, x.view(shape), again, t)) == 0
        assert torch.equal(again.view(6, 8), q) and torch.equal(t.view(6), s)
    for shape in ((8, 6), (48, 1), (1, 48), (2, 4, 6)):
        assert api._call.call(lib.quantize_rows_f32_exo._fast, (None, 6, 8, x.view(shape), q, s)) == -1


@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_tensors_without_memory(lib, name):
    """A meta tensor has an address of zero, which an optional operand would take for None."""
    import torch

    ops = operands(name, SIZES[name])
    for i, o in enumerate(ops):
        meta = torch.ones(o.shape, dtype={"uint16": torch.bfloat16}.get(str(o.dtype), getattr(torch, str(o.dtype))),
                          device="meta")
        with pytest.raises(ValueError, match=f"operand {i + 1} has no memory"):
            getattr(lib, name)(None, *SIZES[name], *ops[:i], meta, *ops[i + 1:])


@pytest.mark.gpu
def test_wrapper_refuses_a_bias_without_memory(lib):
    """The same beside operands on the GPU, where the compiled path makes the calls."""
    import torch

    a, s = torch.ones(3, 5, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
    c = torch.zeros(3, 3, device="cuda")
    lib.gemm_i8_scaled_f32_exo(None, 3, 3, 5, a, a, s, s, None, c)
    c.zero_()
    with pytest.raises(ValueError, match="operand 5 has no memory"):
        lib.gemm_i8_scaled_f32_exo(None, 3, 3, 5, a, a, s, s, torch.ones(3, device="meta"), c)
    assert not c.any()


@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_numbers_beyond_64_bits(lib, name):
    """2^64 is 0 in 64 bits: an activation of that number was SiLU."""
    import torch

    ops = operands(name, SIZES[name])
    for i, size in enumerate(SIZES[name]):
        for wrong in (size + 2 ** 64, size - 2 ** 64, 2 ** 63, -2 ** 63 - 1):
            with pytest.raises(ValueError, match="out of range"):
                getattr(lib, name)(None, *SIZES[name][:i], wrong, *SIZES[name][i + 1:], *ops)
    if torch.cuda.is_available():
        return
    import exo_b200

    with pytest.raises(exo_b200.ExoB200Error):  # any integer type will do otherwise
        getattr(lib, name)(None, *(np.int32(s) for s in SIZES[name]), *ops)


@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_to_write_read_only_arrays(lib, name):
    """Results do not go into arrays that numpy itself would not write (a file mapped for reading, a view of bytes);
    inputs may be such."""
    import torch

    import exo_b200

    first_output = {"quantize_rows": 1, "gemm_i8_scaled": 5, "linear_i8": 4, "gated_bf16_exo": 3,
                    "gated_bf16_backward_exo": 6, "gated_i8_bf16_exo": 6}
    first = next(v for k, v in first_output.items() if name.startswith(k))
    ops = operands(name, SIZES[name])
    for i, o in enumerate(ops):
        fixed = np.frombuffer(o.tobytes(), o.dtype).reshape(o.shape)
        assert not fixed.flags.writeable
        args = (None, *SIZES[name], *ops[:i], fixed, *ops[i + 1:])
        if i >= first:
            with pytest.raises(ValueError, match=f"operand {i + 1} is written"):
                getattr(lib, name)(*args)
        elif not torch.cuda.is_available():
            with pytest.raises(exo_b200.ExoB200Error):  # past the wrapper: there is no device
                getattr(lib, name)(*args)
        assert (fixed == 1).all()


# ------------------------------------------------------------------ contexts and threads
class RecordingLibrary:
    """Stands for the library: remembers on which stream each call would have run."""

    def __init__(self):
        self.context_stream, self.default_stream, self.calls = None, None, []

    def exo_b200_context_set_stream(self, handle, stream):
        import time

        self.context_stream = stream
        time.sleep(0.002)  # another thread's chance

    def exo_b200_set_default_stream(self, stream):
        self.default_stream = stream

    def exo_b200_last_error(self):
        return 0

    def exo_b200_context_destroy(self, handle):
        pass

    def __getattr__(self, name):
        def call(ctx, *args):
            self.calls.append((args[0], self.context_stream if ctx else self.default_stream))

        return call


def recording(monkeypatch, wrapper, name):
    """(library, context, f(context, stream, mark)) with a wrapper whose operands claim to be on a GPU."""
    import ctypes
    import threading

    import torch

    import exo_b200
    from exo_b200 import api

    class OnDevice(torch.Tensor):
        is_cuda = property(lambda self: True)
        __module__ = "torch"  # what the wrapper without checks goes by

    current, dll = threading.local(), RecordingLibrary()
    monkeypatch.setattr(api, "_sync_stream_for", lambda args: current.stream)
    monkeypatch.setattr(api, "_last_default_stream", threading.local())
    context = exo_b200.Context.__new__(exo_b200.Context)
    context.lock, context.handle, context._dll = threading.Lock(), 7, dll
    proc = wrapper(dll, name)

    def make(ctx, stream, mark):
        current.stream = stream
        shapes = {"quantize_rows_f32_exo": ((mark, 2), (mark, 2), (mark,)), "gemm_bf16_exo": ((mark, 2), (2, 2), (mark, 2))}
        types = {"quantize_rows_f32_exo": (torch.float32, torch.int8, torch.float32), "gemm_bf16_exo": (torch.bfloat16,) * 3}
        ops = [torch.zeros(s, dtype=t).as_subclass(OnDevice) for s, t in zip(shapes[name], types[name])]
        proc(ctx, *((mark, 2) if len(proc._argtypes) == 6 else (mark, 2, 2)), *ops)

    return dll, context, make


@pytest.mark.parametrize("wrapper,name", [("CheckedProc", "quantize_rows_f32_exo"), ("ProcWrapper", "gemm_bf16_exo")])
def test_threads_that_share_a_context_keep_their_streams(monkeypatch, wrapper, name):
    """Host threads may share a context: setting its stream and the call are one step."""
    import threading

    from exo_b200 import api

    dll, context, make = recording(monkeypatch, getattr(api, wrapper), name)
    threads = [threading.Thread(target=lambda i=i: [make(context, 1000 + i, i) for _ in range(20)]) for i in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(dll.calls) == 60 and all(stream == 1000 + mark for mark, stream in dll.calls)


@pytest.mark.parametrize("wrapper,name", [("CheckedProc", "quantize_rows_f32_exo"), ("ProcWrapper", "gemm_bf16_exo")])
def test_a_closed_context_is_the_default_one_on_the_callers_stream(monkeypatch, wrapper, name):
    from exo_b200 import api

    dll, context, make = recording(monkeypatch, getattr(api, wrapper), name)
    make(None, 11, 1)
    make(context, 22, 2)
    context.close()
    make(context, 33, 3)
    assert dll.calls == [(1, 11), (2, 22), (3, 33)]


@pytest.mark.gpu
def test_threads_share_a_context(lib):
    """Two host threads, each on its own stream with its own operands, through one explicit context."""
    import threading

    import torch

    import exo_b200

    M, F, K = 50, 333, 257
    wg, wu = (torch.randn(F, K, device="cuda").bfloat16() for _ in range(2))
    want, got, failed = [], [], []
    ctx = exo_b200.Context()
    sources = [torch.randn(M, K, device="cuda").bfloat16() for _ in range(2)]
    for x in sources:
        want.append(torch.zeros(M, F, dtype=torch.bfloat16, device="cuda"))
        got.append([torch.zeros(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(50)])
        lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, want[-1], None, None)
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for o in got[i]:
                    x = sources[i] * 1  # written on this thread's stream just before the call reads it
                    lib.gated_bf16_exo(ctx, 0, M, F, K, x, wg, wu, o, None, None)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)
