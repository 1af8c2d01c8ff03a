"""The AdamW entries without a GPU: the reference's roundings against themselves, the C structure, refusals (nothing falls back to the CPU)."""
import ctypes as C
import os
import re
import subprocess
import sys
import weakref

import numpy as np
import pytest

import adamw_reference as ref
import stochqn_amd
from stochqn_amd import adamw

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_setup_structure_is_the_header_s(tmp_path):
    names = [n for n, _ in adamw._Setup._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include "stochqn_hip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu", sizeof(stochqn_hip_adamw_setup));\n'
                   + "".join('printf(" %%zu", offsetof(stochqn_hip_adamw_setup, %s));\n' % n for n in names) + "return 0;}\n")
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()]
    assert got == [C.sizeof(adamw._Setup)] + [getattr(adamw._Setup, n).offset for n in names]


@pytest.mark.parametrize("torch_is_there", [False, True])
def test_a_star_import_needs_no_torch(torch_is_there):
    """The free-mode objects do without torch, under every import; the objects over tensors come with it."""
    code = ("import sys\n"
            "class No:\n"
            "    def find_spec(self, name, path=None, target=None):\n"
            "        if name.split('.')[0] == 'torch':\n"
            "            raise ModuleNotFoundError(name)\n"
            "    def invalidate_caches(self):\n"
            "        pass\n"
            "%s"
            "from stochqn_amd import *\n"
            "assert oLBFGS_free and SQN_free and adaQN_free and lib and cdll\n"
            "assert ('AdamW_free' in globals()) == ('TensorList' in globals()) == %s\n")
    subprocess.check_call([sys.executable, "-c", code % ("" if torch_is_there else "sys.meta_path.insert(0, No())\n", torch_is_there)], cwd=ROOT)


def test_no_gpu_or_no_device_memory_is_refused(capfd):
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        stochqn_amd.TensorList([torch.zeros(3)])
    with pytest.raises(ValueError):
        stochqn_amd.AdamW_free([torch.zeros(3)])
    lib = adamw._library()
    x = np.zeros(8, dtype=np.float32)
    assert lib.stochqn_hip_tensors_create(1, (C.c_void_p * 1)(x.ctypes.data), (C.c_size_t * 1)(8), (C.c_int * 1)(0)) is None
    assert lib.stochqn_hip_tensors_norm(None, 1.0, 1.0, None, None, None) == -1000
    assert lib.stochqn_hip_tensors_rebind(None, None) == -1000
    assert lib.stochqn_hip_adamw_create(None, None) is None
    assert lib.stochqn_hip_adamw_step(None, None, 0.1, None, None, None) == -1000
    assert lib.stochqn_hip_tensors_state(None, None) == 0 and lib.stochqn_hip_tensors_norm_work(None) == 0
    lib.stochqn_hip_tensors_destroy(None)
    lib.stochqn_hip_adamw_destroy(None)
    err = capfd.readouterr().err
    assert "no usable HIP device" in err or "not device memory" in err
    assert "stochqn_hip_adamw_step: an argument is NULL" in err


@pytest.mark.parametrize("eps", [0.0, 1e-39, 2.0 ** 126 * (1 + 2.0 ** -23), 2e38, float("inf"), float("nan")])
def test_an_eps_that_the_step_cannot_divide_by_is_refused(eps):
    torch = pytest.importorskip("torch")
    with pytest.raises(AssertionError):
        stochqn_amd.AdamW_free([torch.zeros(3)], eps=eps)


@pytest.mark.parametrize("which", ["m", "v"])
def test_the_reference_rounds_to_a_neighbour_and_keeps_the_mean(which):
    """encode then decode: within one step of the code, exact for what the format holds, the mean of many words the value itself."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(128 * 64) * 10.0 ** rng.uniform(-6, 0, 128 * 64)).astype(np.float32)
    if which == "v":
        x = x * x
    word = rng.integers(0, 2 ** 32, x.size, dtype=np.uint64)
    code, byte = ref.encode(x, word, which)
    y = ref.decode(code, byte, which)
    mant = ref.FORMATS[which][0]
    least = np.repeat(2.0 ** (byte.astype(float) - 127), 128) * 2.0 ** (1 - ref.FORMATS[which][1] - mant)
    assert (np.abs(y - x) <= np.maximum(2.0 ** -mant * np.abs(x), least)).all()
    again, same = ref.encode(y.astype(np.float32), word, which)
    kept = np.repeat(same == byte, 128)                     # (the largest may have been rounded up to the next power of two)
    assert kept.mean() > 0.9 and (ref.decode(again, same, which) == y)[kept].all()
    if which == "v":
        assert (y[x > 0] > 0).all()
    # one value, all words: the mean is exact to the words' grain
    block = np.full(128, 1.0, dtype=np.float32)
    block[1:] = np.float32(0.7071)
    total, k = 0.0, 4000
    for i in range(k):
        code, byte = ref.encode(block, np.full(128, (i * 2654435761) % 2 ** 32, dtype=np.uint64), which)
        total += ref.decode(code, byte, which)[5]
    assert abs(total / k - np.float64(block[5])) <= 2.0 ** -mant * 3 / k      # an evenly spread sequence of words: off by a few of k


def test_the_words_are_uniform():
    low, high = ref.words(0, 1 << 18, 12345, 7)
    for w in (low, high, (low & np.uint32(0xFFFF)) << np.uint32(16)):
        counts = np.bincount(w >> np.uint32(26), minlength=64)
        expect = low.size / 64
        assert ((counts - expect) ** 2 / expect).sum() < 64 + 6 * np.sqrt(2 * 64)       # evener than chance is fine, six sigma above is not
    again, _ = ref.words(0, 1 << 18, 12345, 8)
    assert abs(np.corrcoef(low.astype(float), again.astype(float))[0, 1]) < 6 / np.sqrt(low.size)
    part, _ = ref.words(1000, 77, 12345, 7)
    assert (part == low[1000:1077]).all()


class Recorded:
    """Stands for an array of the state: which streams its memory was kept for."""

    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream)


def bare_optimizer(torch, **attributes):
    """An AdamW_free without a GPU: its attributes are what is given, its library answers 0."""
    class Library:
        def stochqn_hip_adamw_step(self, *args):
            return 0

        def stochqn_hip_adamw_destroy(self, handle):
            pass

    class List:
        device, _handle = torch.device("cuda", 0), 1

    opt = object.__new__(adamw.AdamW_free)
    opt.m, opt.v, opt.count, opt._work = (Recorded() for _ in range(4))
    opt.m_scale = opt.v_scale = opt.master = None
    opt._lib, opt._handle, opt.params, opt.gradient, opt._versioned, opt._on, opt._streams = Library(), 1, List(), List(), [], 10, {10}
    for k, v in attributes.items():
        setattr(opt, k, v)
    return opt


def test_a_stream_that_was_first_used_in_a_capture_is_recorded_at_its_first_eager_step(monkeypatch):
    torch = pytest.importorskip("torch")
    opt = bare_optimizer(torch)
    now = {"stream": 10, "capturing": False}
    monkeypatch.setattr(adamw, "_stream", lambda index: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now["stream"])
    for stream, capturing, recorded in ((10, False, []), (20, True, []), (20, True, []), (20, False, [20]), (20, False, [20]), (10, False, [20]), (20, True, [20]),
                                        (30, True, [20]), (20, False, [20]), (30, False, [20, 30]), (10, True, [20, 30]), (30, False, [20, 30])):
        now.update(stream=stream, capturing=capturing)
        opt.run_optimizer(0.1)
        assert all(t.streams == recorded for t in (opt.m, opt.v, opt.count, opt._work)), (stream, capturing)


def test_the_gradients_live_as_long_as_the_step_that_reads_them():
    """Another thread names other gradients while a step is in the library, which has let go of Python's lock: the list that the step was given stays."""
    torch = pytest.importorskip("torch")
    opt = bare_optimizer(torch)
    alive = weakref.ref(opt.gradient)

    class Library(type(opt._lib)):
        def stochqn_hip_adamw_step(self, *args):
            opt.update_gradient(None)                       # as the other thread does
            assert alive() is not None
            return 0

    opt._lib = Library()
    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(adamw, "_stream", lambda index: 10)
        opt.run_optimizer(0.1)
    assert alive() is None and opt.gradient is None


def test_a_state_of_other_shapes_or_types_is_refused_as_a_whole():
    """Arrays that a copy would spread over the optimizer's, or cast: refused in front of the first copy."""
    torch = pytest.importorskip("torch")

    def optimizer(fill):
        sizes = type("Sizes", (), {"sizes": [200]})()
        return bare_optimizer(torch, params=sizes, m=torch.full((256,), fill), v=torch.full((256,), fill), count=torch.full((2,), int(fill)), beta1=0.9, beta2=0.999,
                              eps=1e-8, weight_decay=0.0, state_bits=32, stochastic=False, seed=0, decay=None)
    mine, other = optimizer(1.0), optimizer(2.0)
    good = other.state_dict()
    for name in ("m", "v", "count"):
        for bad in (good[name][:1], good[name].view(2, -1), good[name].to(torch.float16), None, 2.0):
            with pytest.raises(ValueError):
                mine.load_state_dict(dict(good, **{name: bad}))
            assert mine.m.eq(1).all() and mine.v.eq(1).all() and mine.count.eq(1).all(), (name, bad)
    mine.load_state_dict(good)
    assert mine.m.eq(2).all() and mine.v.eq(2).all() and mine.count.eq(2).all()


def test_a_list_of_empty_tensors_belongs_to_their_device(monkeypatch):
    """The library looks at no address of an empty tensor: a list of nothing else is made while the tensors' device is the current one."""
    torch = pytest.importorskip("torch")
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, current[0] = current[0], torch.device(self.index).index if not isinstance(self.index, int) else self.index

        def __exit__(self, *args):
            current[0] = self.was

    class Library:
        def stochqn_hip_tensors_create(self, *args):
            self.on = current[0]
            return 1

        def stochqn_hip_tensors_norm_work(self, handle):
            return 1

        def stochqn_hip_tensors_destroy(self, handle):
            pass

    class Empty:
        dtype, is_cuda, device, layout = torch.float32, True, torch.device("cuda", 1), torch.strided
        get_device, numel, data_ptr = lambda self: 1, lambda self: 0, lambda self: 0
        is_contiguous, is_neg, untyped_storage = lambda self: True, lambda self: False, lambda self: None

    library = Library()
    monkeypatch.setattr(adamw, "_library", lambda: library)
    monkeypatch.setattr(torch.cuda, "device", Device)
    adamw.TensorList([Empty(), Empty()])
    assert library.on == 1 and current[0] == 0


@pytest.mark.parametrize("which", ["asan", "tsan"])
def test_the_host_side_under_sanitizers(which):
    """What tensors.cpp hands to the kernels (every element of every tensor in one tile of one launch) and what it refuses, every HIP call failing
    in turn; threads that step, rebind and take the norm of one list at once."""
    here = os.path.join(ROOT, "tests", "hostsim")
    subprocess.check_call(["make", "-C", here, "build/tensors_" + which], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    for args in ([], ["threads"]) if which == "asan" else (["threads"],):
        run = subprocess.run([os.path.join(here, "build", "tensors_" + which)] + args, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr[-3000:]


def kernels_of(asm):
    """name -> basic blocks of every kernel of an assembly listing: (label or None, instructions, labels that may follow), in textual order; a block
    that does not end in an unconditional jump or the program's end falls through to the next."""
    found = {}
    for name, body in re.findall(r"^(_Z\w+):.*?\n(.*?)^\.Lfunc_end", asm, re.M | re.S):
        blocks = [[None, [], [], True]]
        for line in body.splitlines():
            line = line.split(";")[0].strip()
            label = re.match(r"(\.LBB\w+):", line)
            if label:
                blocks.append([label.group(1), [], [], True])
                continue
            if not line or line.startswith("."):
                continue
            op = line.split()[0]
            blocks[-1][1].append(line)
            if op in ("s_branch", "s_endpgm") or op.startswith("s_cbranch"):
                if op != "s_endpgm":
                    blocks[-1][2].append(line.split()[1])
                blocks[-1][3] = op.startswith("s_cbranch")
                blocks.append([None, [], [], True])
            elif op == "s_barrier":                                         # a block of its own end: what follows is behind it
                blocks.append([None, [], [], True])
            assert op not in ("s_setpc_b64", "s_swappc_b64"), line
        found[name] = blocks
    return found


def reached(blocks, start, through):
    at = {b[0]: k for k, b in enumerate(blocks) if b[0]}
    seen, todo = set(), list(start)
    while todo:
        k = todo.pop()
        if k in seen or k >= len(blocks):
            continue
        seen.add(k)
        if through(blocks[k]):
            todo += [at[label] for label in blocks[k][2]] + ([k + 1] if blocks[k][3] else [])
    return seen


def test_a_step_is_counted_behind_a_barrier(tmp_path):
    """Every wave of a workgroup reads the step counter by itself, one thread arrives for all of them and the last to arrive writes it: in the
    compiled kernels every way to an arrival, and to what is stored behind one, leads over a barrier of the workgroup."""
    asm = tmp_path / "tensors.s"
    subprocess.check_call(["make", "-C", os.path.join(ROOT, "stochqn_amd", "csrc"), "device-asm", "ASM=%s" % asm], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    steps = {n: b for n, b in kernels_of(asm.read_text()).items() if "k_adamw" in n}
    assert len(steps) == 6
    for name, blocks in steps.items():
        has = lambda b, what: any(line.startswith(what) for line in b[1])
        arrivals = [k for k, b in enumerate(blocks) if has(b, "global_atomic")]
        assert len(arrivals) == 2, name
        counted = arrivals + [k for k in reached(blocks, arrivals, lambda b: True) if has(blocks[k], "global_store")]
        assert len(counted) >= 5, name                                       # ... the stores that reset both counters, and the count
        early = reached(blocks, [0], lambda b: not has(b, "s_barrier"))
        assert not early & set(counted), name
