"""The AdamW entries without a GPU: the reference's roundings against themselves, the C structure, refusals (nothing falls back to the CPU)."""
import ctypes as C
import os
import subprocess

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


@pytest.mark.parametrize("which", ["asan", "tsan"])
def test_the_host_side_under_sanitizers(which):
    """What tensors.cpp hands to the kernels (every element of every tensor in one tile of one launch) and what it refuses, every HIP call failing
    in turn; threads that step, rebind and take the norm of one list at once."""
    here = os.path.join(ROOT, "tests", "hostsim")
    subprocess.check_call(["make", "-C", here, "build/tensors_" + which], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    for args in ([], ["threads"]) if which == "asan" else (["threads"],):
        run = subprocess.run([os.path.join(here, "build", "tensors_" + which)] + args, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr[-3000:]
