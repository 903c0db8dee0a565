"""The 4-bit cache and log probabilities without a GPU: the library exports what include/fyodor_hip_kv4.h and
include/fyodor_hip_logprobs.h declare, every entry refuses the calls it documents as declined (nothing is enqueued, so
no GPU is needed), and the statements that the GPU tests use keep their own invariants."""
import ctypes
import math

import numpy as np
import pytest

from fyodor_amd import KERNEL_LIBRARY
from fyodor_amd.hip import Kernels, Kv4
from kv4_check import BLOCK, Cache4, held, logprobs, quantised, step_of, store
from test_boundary import declared, exported
from test_serving import BAD_GEOMETRY, refuse

A = 1 << 20   # an aligned address that no refused call looks at


@pytest.fixture(scope="module")
def kernels():
    return Kernels()


def cache(**change):
    return Kv4(**dict(dict(keys=A, values=A, key_steps=A, value_steps=A, pages=64, page_tokens=32, kv_heads=2,
                           width=128), **change))


BAD_ADDRESS = [{"keys": 0}, {"keys": A + 8}, {"values": 0}, {"values": A + 4}, {"key_steps": 0}, {"key_steps": A + 8},
               {"value_steps": 0}, {"value_steps": A + 2}]


def test_library_exports_the_headers():
    want = declared("fyodor_hip_kv4.h")
    assert want == {"nya_hip_kv4_bytes", "nya_hip_kv4_store", "nya_hip_kv4_load", "nya_hip_kv4_attention_bytes",
                    "nya_hip_kv4_attention"}
    answers = declared("fyodor_hip_logprobs.h")
    assert answers == {"nya_hip_logprobs_bytes", "nya_hip_logprobs"}
    assert want | answers <= exported(KERNEL_LIBRARY)


def test_kv4_bytes(kernels):
    assert kernels.kv4_bytes(100, 32, 3, 64) == (100 * 32 * 3 * 32, 100 * 32 * 3 * 4)
    # Past 32 bits.
    assert kernels.kv4_bytes((1 << 24) - 1, 128, 8, 512) == (((1 << 24) - 1) * 128 * 8 * 256,
                                                             ((1 << 24) - 1) * 128 * 8 * 32)
    codes, steps = ctypes.c_size_t(), ctypes.c_size_t()
    for change in BAD_GEOMETRY:
        assert kernels.lib.nya_hip_kv4_bytes(cache(**change), codes, steps) == 1
    assert kernels.lib.nya_hip_kv4_bytes(None, codes, steps) == 1
    assert kernels.lib.nya_hip_kv4_bytes(cache(), None, steps) == 1
    assert kernels.lib.nya_hip_kv4_bytes(cache(), codes, None) == 1


def test_kv4_store_and_load_refusals(kernels):
    far = 1 << 28
    good = dict(cache=cache(), slots=A, count=4, k=A, k_stride=256, v=A, v_stride=256, angles=A, rotated=64, layout=1,
                q=A, q_stride=512, q_out=A + far, q_out_stride=512, heads=4, stream=0)
    refuse(kernels.lib.nya_hip_kv4_store, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] +
           [{"cache": None}, {"slots": 0}, {"slots": A + 1}, {"count": 0}, {"count": (1 << 22) + 1}, {"k": 0},
            {"k": A + 2}, {"v": 0}, {"k_stride": 255}, {"v_stride": 255}, {"v_stride": 1 << 31}, {"angles": A + 4},
            {"angles": 0}, {"rotated": 0}, {"rotated": 33}, {"rotated": 130}, {"layout": 2}, {"q_out": 0},
            {"q_out": A + 16}, {"q_stride": 511}, {"q_out_stride": 511}, {"heads": 0},
            {"k": A + far}, {"v": A + far + 4096}, {"v": A + far - 4}])
    good = dict(cache=cache(), slots=A, count=4, k=A, k_stride=256, v=A + far, v_stride=256, stream=0)
    refuse(kernels.lib.nya_hip_kv4_load, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] +
           [{"cache": None}, {"slots": 0}, {"count": 0}, {"k": 0}, {"v": 0}, {"v": A}, {"v": A + 1024},
            {"k_stride": 255}, {"v_stride": 255}])


def test_kv4_attention_refusals(kernels):
    far = 1 << 28
    good = dict(cache=cache(), q=A, q_stride=512, out=A + far, out_stride=512, count=4, starts=A, lengths=A, table=A,
                table_stride=8, requests=2, max_tokens=4, max_length=100, heads=4, window=0, scale=0.1, workspace=A,
                workspace_bytes=64, stream=0)
    sizes = [{"count": 0}, {"requests": 0}, {"requests": 65536}, {"max_tokens": 0}, {"max_tokens": 5},
             {"max_length": 0}, {"heads": 0}, {"heads": 3}, {"window": 1 << 31}]
    refuse(kernels.lib.nya_hip_kv4_attention, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] + sizes +
           [{"cache": None}, {"q": 0}, {"q": A + 1}, {"out": 0}, {"out": A}, {"out": A + 2048}, {"q_stride": 511},
            {"out_stride": 500}, {"starts": 0}, {"lengths": 0}, {"table": 0}, {"table": A + 3}, {"table_stride": 0},
            {"table_stride": 1 << 31}, {"workspace": A + 8}, {"scale": math.nan}, {"scale": math.inf}])
    b = ctypes.c_size_t()
    good = dict(cache=cache(), count=4, requests=2, max_tokens=4, max_length=100, heads=4, window=0,
                bytes=ctypes.byref(b))
    assert kernels.lib.nya_hip_kv4_attention_bytes(*good.values()) == 0
    refuse(kernels.lib.nya_hip_kv4_attention_bytes, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY] + sizes + [{"cache": None}, {"bytes": None}])


def test_logprobs_refusals(kernels):
    far = 1 << 28
    good = dict(logits=A, stride=1000, n=999, count=7, mask=A + far, scale=1.0, tokens=A + 2 * far,
                logprobs=A + 3 * far, ranks=A + 4 * far, entropies=A + 5 * far, top=5, top_ids=A + 6 * far,
                top_logprobs=A + 7 * far, workspace=A + 8 * far, workspace_bytes=0, stream=0)
    end = A + 4 * (6 * 1000 + 999)
    refuse(kernels.lib.nya_hip_logprobs, good,
           [{"logits": 0}, {"logits": A + 2}, {"stride": 998}, {"stride": 1 << 31}, {"n": 0}, {"n": (1 << 24) + 1,
            "stride": 1 << 25}, {"count": 0}, {"count": (1 << 22) + 1}, {"mask": A + 1}, {"scale": 0.0},
            {"scale": -1.0}, {"scale": math.nan}, {"scale": math.inf}, {"scale": 0.9 * 2.0 ** -20}, {"scale": 1.1 * 2.0 ** 20},
            {"tokens": A + 3}, {"logprobs": 0},
            {"logprobs": A + 3 * far + 2}, {"ranks": A + 1}, {"entropies": A + 2}, {"top": 65}, {"top_ids": 0},
            {"top_logprobs": 0}, {"top_ids": A + 1}, {"top_logprobs": A + 3}, {"workspace": A + 8},
            {"tokens": 0, "entropies": 0, "top": 0},
            # Outputs over inputs and over each other.
            {"logprobs": end - 4}, {"entropies": A - 4}, {"top_ids": A - 4 * 34}, {"ranks": A + 2 * far},
            {"top_logprobs": A + far + 4}, {"entropies": A + 3 * far + 24}, {"ranks": A + 6 * far + 4 * 34},
            {"top_ids": A + 7 * far}])
    b = ctypes.c_size_t()
    assert kernels.lib.nya_hip_logprobs_bytes(999, 7, 5, ctypes.byref(b)) == 0
    for bad in ((0, 7, 5), ((1 << 24) + 1, 7, 5), (9, 0, 5), (9, (1 << 22) + 1, 5), (9, 7, 65)):
        assert kernels.lib.nya_hip_logprobs_bytes(*bad, ctypes.byref(b)) == 1
    assert kernels.lib.nya_hip_logprobs_bytes(9, 7, 5, None) == 1


@pytest.mark.parametrize("n", [1, 984, 2046, 2047, 32000, 50257, 128256, 131070, 262147, 1 << 24])
def test_logprobs_scratch_of_the_largest_batch(kernels, n):
    """Scratch for the largest batch and the most alternatives is what every smaller one wants."""
    said = {(rows, top): kernels.logprobs_bytes(n, rows, top) for rows in range(1, 1100) for top in (0, 1, 64)}
    for top in (0, 1, 64):
        sizes = [said[rows, top] for rows in range(1, 1100)]
        assert sizes == sorted(sizes)
        assert kernels.logprobs_bytes(n, 1 << 22, top) == sizes[-1] <= 20 << 20
    assert all(said[rows, 0] <= said[rows, 1] == said[rows, 64] for rows in range(1, 1100))
    # Rows longer than a tile of 2048 are split while there are few.
    assert (said[1, 0] > 0) == (n > 2045)


def test_steps():
    """Steps by hand: 8 bits, ties to even, the negative one of two extremes, the ends."""
    def block(*x):
        return np.array(list(x) + [0] * (BLOCK - len(x)), np.float32)
    for x, want in [((8,), -1), ((-8,), 1), ((8, -8), 1), ((7.99, -8), 1), ((8.01, -8), -1), ((0,), 0),
                    ((8 * 129.5,), -130), ((8 * 130.5,), -130), ((8 * 131.4999,), -131), ((8 * 255.5,), -256),
                    ((1e30,), -8160), ((-65280,), 8160), ((2.0 ** -21,), -2.0 ** -24), ((2.0 ** -22,), 0),
                    ((2.0 ** -22 * 1.01,), -2.0 ** -24), ((1e-40,), 0)]:
        assert step_of(block(*x)) == np.float16(want), x


@pytest.mark.parametrize("size", [1.0, 1e-6, 3e-7, 1e4, 1e6])
def test_quantised(size):
    """What is held is an fp16 number, off by half a step, or a whole one on the far side."""
    x = (size * np.random.default_rng(1).standard_normal((200, 64))).astype(np.float32)
    codes, steps = quantised(x)
    assert codes.max() <= 15
    d = np.repeat(steps.astype(np.float64), BLOCK, 1)
    got = (codes.astype(np.float64) - 8) * d
    assert np.array_equal(got, got.astype(np.float16).astype(np.float64))
    # The step is off by 2^-8 of itself (in fp16's last places by half of 2^-24), eight of them by 8 times that.
    off = np.abs(got - np.clip(x, -65280, 65280))
    assert np.all(off <= np.abs(d) * (1 + 8 * 2.0 ** -8) + 8 * 2.0 ** -25)
    # (Clamped elements of the far side are 7 steps of 8160, a whole step off, however many they are.)
    inside = np.abs(x) < 57120
    assert np.mean((off <= np.abs(d) * (0.5 + 8 * 2.0 ** -8) + 8 * 2.0 ** -25)[inside]) > 0.95


@pytest.mark.parametrize("exponent", [*range(-26, -9), -3, 0, 5, 14, 15, 16, 20, 60])
def test_off_by_as_declared(exponent):
    """How far what is held may be off, as the header says it, and that it is held the same when stored again. With m
    the largest magnitude, d0 = m / -8 and |d - d0| <= 2^-8 |d0|, in fp16's subnormals 2^-25 more: codes -8 .. 7 leave
    half a step or, past -8 steps, |m| - 8 |d| <= |d| / 32 (1 + 2^-7) + 2^-22; past 7 steps |m| - 7 |d|, one step more
    than that. (A 32nd of a step rounds to (1 + 2^-7) of it; zeros are off by |m| <= 2^-22 (1 + 2^-8).)"""
    rng = np.random.default_rng(exponent + 100)
    x = rng.standard_normal((2000, BLOCK))
    x[::3, 3] = -x[::3, 7] * (1 - rng.random(667) / 16)   # near -m, in some of them
    x[::3, 7] = np.abs(x[::3]).max(1) * np.sign(x[::3, 7])
    x = (x / np.abs(x).max(1, keepdims=True) * 2.0 ** (exponent + rng.random((2000, 1)))).astype(np.float32)
    codes, steps = quantised(x)
    d, y = steps.astype(np.float64), x.astype(np.float64)
    got = (codes.astype(np.float64) - 8) * d
    other = y * d > 0                                     # (m's own side has d's other sign)
    y = np.where(other, np.clip(y, -57120, 57120), np.clip(y, -65280, 65280))
    m = np.abs(x).max(1, keepdims=True)
    more = np.where(m < 2.0 ** -14, 2.0 ** -22 * (1 + 2.0 ** -8), 0)
    bound = np.abs(d) * np.where(other, 1 + (1 + 2.0 ** -7) / 32, 0.5) + more
    assert np.all(np.abs(got - y) <= bound)
    assert np.all(bound[(m >= 2.0 ** -14).ravel()] <= (m / np.where(other, 7.5, 15.8))[(m >= 2.0 ** -14).ravel()])
    assert not got[(m <= 2.0 ** -22).ravel()].any()
    again = quantised(got.astype(np.float32))
    whole = (m >= 2.0 ** -14).ravel()
    assert np.array_equal(again[0][whole], codes[whole]) and np.array_equal(again[1][whole], steps[whole])


@pytest.mark.parametrize("page_tokens,width", [(16, 64), (32, 128), (128, 256), (64, 512)])
def test_layout(page_tokens, width):
    """Every nibble and every step has its own place, and the statement stores and reads back."""
    rng = np.random.default_rng(width)
    k, v = (Cache4(3, page_tokens, 2, width, rng, kind) for kind in "kv")
    for c in (k, v):
        at, shift = c._places()
        places = (2 * at + (shift > 0)).ravel()
        assert np.array_equal(np.sort(places), np.arange(page_tokens * width))
        assert np.array_equal(np.sort(c._step_places().ravel()), np.arange(page_tokens * width // BLOCK))
        assert np.array_equal(c.unpack(c.packed()), c.codes)
        assert np.array_equal(c.unpack_steps(c.packed_steps()).view(np.uint16), c.steps.view(np.uint16))
    x = rng.standard_normal((2, 2, 2, width)).astype(np.float32)
    x[0, 1, 1, 3] = np.inf
    store(k, v, [page_tokens + 5, -1], x[0], x[1])
    a, b = held(k, v)
    assert np.all(np.abs(a[1, 0, 5] - x[0, 0, 0]) < 0.5) and np.all(np.abs(b[1, :, 5] - x[1, 0]) < 0.5)
    store(k, v, [3 * page_tokens - 1, 7], x[0][::-1], x[1])
    a, b = held(k, v)
    assert np.isnan(a[2, 1, -1]).all() and np.isnan(b[2, 1, -1]).all() and np.isfinite(b[2, 0, -1]).all()


def test_logprobs_statement():
    x = np.array([[1, 3, 3, -np.inf, 2], [0, np.nan, 0, 0, 0], [-np.inf] * 5], np.float32)
    lp, ranks, entropy, ids, top, _ = logprobs(x, None, 1.0, [2, 0, 0], 5)
    p = np.exp([1, 3, 3, 2]) / np.exp([1, 3, 3, 2]).sum()
    assert ranks.tolist() == [1, -1, -1] and ids[0].tolist() == [1, 2, 4, 0, -1] and (ids[1:] == -1).all()
    assert math.isclose(lp[0], math.log(p[2])) and math.isclose(entropy[0], -(p * np.log(p)).sum())
    assert top[0, 4] == -np.inf and np.isnan(top[1:]).all() and np.isnan(lp[1:]).all()
    assert logprobs(x, np.array([2], np.uint32), 1.0, [1, 0, 9], 1)[0][:2].tolist()[0] == -np.inf
