"""The serving part of the kernel library without a GPU: the library exports
what include/fyodor_hip_serving.h declares, every entry refuses the calls
it documents as declined (nothing is enqueued, so no GPU is needed), the
rotary frequencies follow their formulas, and the numpy statement of the page
step that the GPU tests use keeps its own invariants."""
import ctypes
import math

import numpy as np
import pytest

from fyodor_amd import KERNEL_LIBRARY
from fyodor_amd.hip import Kernels, Kv8
from serving_check import F32_HALF, Pages, bands
from test_boundary import declared, exported

A = 1 << 20   # an aligned address that no refused call looks at


@pytest.fixture(scope="module")
def kernels():
    return Kernels()


def test_library_exports_the_serving_header():
    want = declared("fyodor_hip_serving.h")
    assert want == {"nya_hip_page_step", "nya_hip_rope_frequencies", "nya_hip_rope_angles", "nya_hip_rope",
                    "nya_hip_kv8_bytes", "nya_hip_kv8_store", "nya_hip_kv8_load", "nya_hip_kv8_attention_bytes",
                    "nya_hip_kv8_attention"}
    assert want <= exported(KERNEL_LIBRARY)


def refuse(call, good, changes):
    """Every change to the good arguments (never made themselves) is declined with 1."""
    for change in changes:
        args = dict(good, **change)
        assert call(*args.values()) == 1, change


def test_page_step_refusals(kernels):
    good = dict(lengths=A, counts=A, requests=4, page_tokens=16, table=A, table_stride=8, held=A, free_pages=A,
                pages=64, free_count=A, starts=A, positions=A, slots=A, max_tokens=8, stream=0)
    names = ["lengths", "counts", "table", "held", "free_pages", "free_count", "starts", "positions", "slots"]
    refuse(kernels.lib.nya_hip_page_step, good,
           [{n: v} for n in names for v in (0, A + 2)] +
           [{"requests": 0}, {"requests": 65537}, {"page_tokens": 0}, {"page_tokens": 24}, {"page_tokens": 256},
            {"table_stride": 0}, {"table_stride": 1 << 30}, {"requests": 65536, "table_stride": 1 << 15}, {"pages": 0},
            {"pages": 1 << 28}, {"max_tokens": 0}, {"max_tokens": (1 << 22) + 1}])


def test_rope_refusals(kernels):
    L = kernels.lib
    refuse(L.nya_hip_rope_angles, dict(positions=A, count=3, frequencies=A, rotated=64, magnitude=1.0, angles=A,
                                       stream=0),
           [{"positions": 0}, {"positions": A + 1}, {"frequencies": 0}, {"angles": 0}, {"angles": A + 4}, {"count": 0},
            {"count": (1 << 22) + 1}, {"rotated": 0}, {"rotated": 63}, {"rotated": 1026}, {"magnitude": math.inf},
            {"magnitude": math.nan}])
    far = 1 << 28
    good = dict(q=A, q_stride=512, q_out=A + far, q_out_stride=512, heads=4, k=A + 2 * far, k_stride=256,
                k_out=A + 3 * far, k_out_stride=256, kv_heads=2, width=128, count=5, angles=A, rotated=64, layout=0,
                stream=0)
    refuse(L.nya_hip_rope, good,
           [{"q": 0}, {"q": A + 2}, {"q_out": 0}, {"q_out": A + 4}, {"q_out": A, "q_out_stride": 516},
            {"q_stride": 511}, {"q_out_stride": 511}, {"heads": 0}, {"heads": 65536}, {"width": 0},
            {"width": 1 << 23}, {"k_out": 0}, {"k_out": A + 2 * far + 4}, {"k_stride": 255}, {"kv_heads": 0},
            {"count": 0}, {"count": (1 << 22) + 1}, {"angles": 0}, {"angles": A + 4}, {"rotated": 0}, {"rotated": 65},
            {"rotated": 130}, {"layout": 2}])


def test_rope_frequency_refusals(kernels):
    out, mag = np.empty(64, np.float32), ctypes.c_float()
    good = dict(out=out.ctypes.data, rotated=128, base=10000.0, factors=None, scaling=3, factor=4.0, original=4096.0,
                low=1.0, high=32.0, magnitude=ctypes.byref(mag))
    assert kernels.lib.nya_hip_rope_frequencies(*good.values()) == 0
    refuse(kernels.lib.nya_hip_rope_frequencies, good,
           [{"out": None}, {"magnitude": None}, {"rotated": 0}, {"rotated": 127}, {"base": 1.0}, {"base": math.nan},
            {"base": math.inf}, {"scaling": 4}, {"factor": 0.5}, {"factor": math.nan}, {"factor": math.inf},
            {"original": 0.0}, {"original": math.inf}, {"low": 0.0}, {"low": 32.0}, {"high": math.inf},
            {"scaling": 2, "low": -1.0}])


@pytest.mark.parametrize("rotated,base", [(2, 10000.0), (64, 500000.0), (128, 10000.0), (512, 1000000.0)])
def test_rope_frequencies(kernels, rotated, base):
    j = np.arange(rotated // 2)
    plain = base ** (-2.0 * j / rotated)
    # pow and the divisions are off by a few steps of 64 bits.
    close = lambda got, want: np.all(np.abs(got - want) <= want * F32_HALF * (1 + 1e-6))
    f, m = kernels.rope_frequencies(rotated, base)
    assert m == 1 and close(f, plain)
    f, m = kernels.rope_frequencies(rotated, base, scaling="linear", factor=8.0)
    assert m == 1 and close(f, plain / 8)
    factors = np.linspace(1, 9, rotated // 2).astype(np.float32)
    f, m = kernels.rope_frequencies(rotated, base, factors=factors)
    assert m == 1 and close(f, plain / factors)
    f, m = kernels.rope_frequencies(rotated, base, scaling="bands", factor=8.0, original=8192, low=1, high=4)
    assert m == 1 and close(f, bands(rotated, base, 8.0, 8192, 1, 4))
    f, m = kernels.rope_frequencies(rotated, base, scaling="ramp", factor=4.0, original=4096, low=1, high=32)
    pair = lambda turns: rotated * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(base))
    first, last = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rotated - 1)
    g = 1 - np.clip((j - first) / max(last - first, 1e-3), 0, 1)
    assert abs(m - (1 + 0.1 * math.log(4))) <= 2 * F32_HALF and close(f, g * plain + (1 - g) * plain / 4)
    # A factor of 1 changes nothing, whatever the form.
    for scaling in ("linear", "bands", "ramp"):
        f, m = kernels.rope_frequencies(rotated, base, scaling=scaling, factor=1.0, original=4096, low=1, high=32)
        assert m == 1 and np.all(np.abs(f - plain) <= plain * F32_HALF * 2.001)


def cache(**change):
    return Kv8(**dict(dict(keys=A, values=A, key_scales=A, value_scales=A, pages=64, page_tokens=32, kv_heads=2,
                           width=128), **change))


BAD_GEOMETRY = [{"pages": 0}, {"pages": 1 << 26}, {"pages": 1 << 25, "kv_heads": 64}, {"page_tokens": 8},
                {"page_tokens": 48}, {"page_tokens": 256}, {"kv_heads": 0}, {"kv_heads": 65536}, {"width": 0},
                {"width": 96}, {"width": 1024}]
BAD_ADDRESS = [{"keys": 0}, {"keys": A + 8}, {"values": 0}, {"values": A + 4}, {"key_scales": 0},
               {"key_scales": A + 2}, {"value_scales": 0}]


def test_kv8_bytes(kernels):
    assert kernels.kv8_bytes(100, 32, 3, 64) == (100 * 32 * 3 * 64, 1200)
    # Past 32 bits.
    assert kernels.kv8_bytes((1 << 24) - 1, 128, 8, 512) == (((1 << 24) - 1) * 128 * 8 * 512, ((1 << 24) - 1) * 32)
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    for change in BAD_GEOMETRY:
        assert kernels.lib.nya_hip_kv8_bytes(cache(**change), codes, scales) == 1
    assert kernels.lib.nya_hip_kv8_bytes(None, codes, scales) == 1
    assert kernels.lib.nya_hip_kv8_bytes(cache(), None, scales) == 1
    assert kernels.lib.nya_hip_kv8_bytes(cache(), codes, None) == 1


def test_kv8_store_and_load_refusals(kernels):
    far = 1 << 28
    good = dict(cache=cache(), slots=A, count=4, k=A, k_stride=256, v=A, v_stride=256, angles=A, rotated=64, layout=1,
                q=A, q_stride=512, q_out=A + far, q_out_stride=512, heads=4, stream=0)
    refuse(kernels.lib.nya_hip_kv8_store, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] +
           [{"cache": None}, {"slots": 0}, {"slots": A + 1}, {"count": 0}, {"count": (1 << 22) + 1}, {"k": 0},
            {"k": A + 2}, {"v": 0}, {"k_stride": 255}, {"v_stride": 255}, {"v_stride": 1 << 31}, {"angles": A + 4},
            {"angles": 0}, {"rotated": 0}, {"rotated": 33}, {"rotated": 130}, {"layout": 2}, {"q_out": 0},
            {"q_out": A + 16}, {"q_stride": 511}, {"q_out_stride": 511}, {"heads": 0}])
    good = dict(cache=cache(), slots=A, count=4, k=A, k_stride=256, v=A + far, v_stride=256, stream=0)
    refuse(kernels.lib.nya_hip_kv8_load, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] +
           [{"cache": None}, {"slots": 0}, {"count": 0}, {"k": 0}, {"v": 0}, {"v": A}, {"v": A + 1024},
            {"k_stride": 255}, {"v_stride": 255}, {"k_stride": 511, "v_stride": 511, "v": A + 1024},
            {"k_stride": 768, "v_stride": 768, "v": A + 1020}])


def test_rows_that_overlap(kernels):
    """A row that a call writes is no other row's input or output; parts of common rows are apart."""
    far, L = 1 << 28, kernels.lib
    rope = dict(q=A, q_stride=512, q_out=A + far, q_out_stride=512, heads=4, k=A + 2 * far, k_stride=256,
                k_out=A + 3 * far, k_out_stride=256, kv_heads=2, width=128, count=5, angles=A, rotated=64, layout=0,
                stream=0)
    refuse(L.nya_hip_rope, rope,
           [{"k": A + far}, {"k": A + far + 2048}, {"k_out": A + far + 4 * 2047}, {"k": A + far, "k_out": A + far},
            {"k": A, "k_out": A}, {"k": A + 2044, "k_stride": 512, "k_out": A, "q_out": A, "k_out_stride": 512},
            # q | k in common rows of 768 in place, k one float too early
            {"q_out": A, "q_stride": 768, "q_out_stride": 768, "k": A + 2044, "k_out": A + 2044, "k_stride": 768,
             "k_out_stride": 768}])
    store = dict(cache=cache(), slots=A, count=4, k=A + 2 * far, k_stride=256, v=A + 3 * far, v_stride=256, angles=A,
                 rotated=64, layout=1, q=A, q_stride=512, q_out=A + far, q_out_stride=512, heads=4, stream=0)
    refuse(L.nya_hip_kv8_store, store,
           [{"k": A + far}, {"v": A + far + 4096}, {"v": A + far - 4}, {"q_out": A + 2 * far}, {"q_out": A + 3 * far - 4}])


def test_kv8_attention_refusals(kernels):
    far = 1 << 28
    good = dict(cache=cache(), q=A, q_stride=512, out=A + far, out_stride=512, count=4, starts=A, lengths=A, table=A,
                table_stride=8, requests=2, max_tokens=4, max_length=100, heads=4, window=0, scale=0.1, workspace=A,
                workspace_bytes=64, stream=0)
    sizes = [{"count": 0}, {"requests": 0}, {"requests": 65536}, {"max_tokens": 0}, {"max_tokens": 5},
             {"max_length": 0}, {"heads": 0}, {"heads": 3}, {"window": 1 << 31}]
    refuse(kernels.lib.nya_hip_kv8_attention, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY + BAD_ADDRESS] + sizes +
           [{"cache": None}, {"q": 0}, {"q": A + 1}, {"out": 0}, {"out": A}, {"out": A + 2048}, {"q_stride": 511},
            {"out_stride": 500}, {"starts": 0}, {"lengths": 0}, {"table": 0}, {"table": A + 3}, {"table_stride": 0},
            {"table_stride": 1 << 31}, {"workspace": A + 8}, {"scale": math.nan}, {"scale": math.inf}])
    b = ctypes.c_size_t()
    good = dict(cache=cache(), count=4, requests=2, max_tokens=4, max_length=100, heads=4, window=0,
                bytes=ctypes.byref(b))
    assert kernels.lib.nya_hip_kv8_attention_bytes(*good.values()) == 0
    refuse(kernels.lib.nya_hip_kv8_attention_bytes, good,
           [{"cache": cache(**c)} for c in BAD_GEOMETRY] + sizes + [{"cache": None}, {"bytes": None}])


def test_kv8_attention_limits(kernels):
    """The largest steps are answered, larger ones declined; empty places do not make the workspace large."""
    def ask(count, requests, heads, kv_heads, width=128, max_tokens=1, max_length=4096):
        b = ctypes.c_size_t()
        done = kernels.lib.nya_hip_kv8_attention_bytes(cache(kv_heads=kv_heads, width=width), count, requests,
                                                       max_tokens, max_length, heads, 0, ctypes.byref(b))
        return done, b.value
    assert ask(1 << 22, 1, 32, 8, max_tokens=1 << 22)[0] == 0
    assert ask(1 << 22, 1, 33, 3)[0] == 1
    assert ask(1 << 22, 1, 33, 3, width=512)[0] == 1
    assert ask(65535, 65535, 32, 32)[0] == 0
    assert ask(65535, 65535, 33, 33)[0] == 1
    # A prompt of 600 tokens somewhere among 65535 requests.
    for width in (64, 128, 256, 512):
        done, size = ask(700, 65535, 32, 32, width, max_tokens=600)
        assert done == 0 and size < 1 << 32


@pytest.mark.parametrize("seed", range(4))
def test_page_statement(seed):
    """The statement the GPU is held to: no page is held twice or lost, and every slot is its request's."""
    rng = np.random.default_rng(seed)
    size, pages, requests = 16, 40, 7
    state = Pages(requests, 12, pages, size, rng.permutation(pages))
    for _ in range(30):
        lengths = rng.integers(0, 12 * size + 20, requests)
        counts = np.minimum(rng.integers(0, 40, requests), lengths)
        starts, positions, slots = state.step(lengths, counts, 200)
        live = [state.table[r, j] for r in range(requests) for j in range(state.held[r])]
        assert sorted(live + state.free_pages[:state.free_count[0]].tolist()) == list(range(pages))
        for r in range(requests):
            assert np.all(state.table[r, state.held[r]:] == -1)
            for row in range(starts[r], starts[r + 1]):
                if slots[row] >= 0:
                    assert state.table[r, positions[row] // size] == slots[row] // size
                    assert slots[row] % size == positions[row] % size
