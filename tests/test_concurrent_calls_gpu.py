"""Operators that make several launches in one call, called by several threads at once: on one handle and one stream, whose scratch they share."""
import threading

import numpy as np
import pytest

import helium_amd as ha
from device_arrays import Array, empty
from gradient_clip_cases import inputs as clip_inputs
from int8_cases import inputs as int8_inputs
from rms_norm_cases import EPSILON
from rms_norm_cases import inputs as norm_inputs

pytestmark = pytest.mark.gpu

THREADS, CALLS = 4, 15


def at_once(calls):
    """Each of `calls` CALLS times, by a thread of its own."""
    failed = []

    def repeat(call):
        try:
            for _ in range(CALLS):
                call()
        except Exception as e:  # noqa: BLE001 (told to the main thread)
            failed.append(e)

    threads = [threading.Thread(target=repeat, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ha.device.synchronize()
    assert not failed, failed


def test_gradients_of_the_norm(gpu):
    rows, columns = 3000, 515
    norm = ha.RmsNorm(columns, "f32", epsilon=EPSILON)
    calls, results = [], []
    for k in range(THREADS):
        host, _ = norm_inputs(rows, columns, "f32", None, "f32", seed=k)
        operands = [Array(host[n]) for n in ("dy", "h", "gamma", "rstd")] + [empty((rows, columns), np.float32), empty((columns,), np.float32)]
        call = lambda o=operands: norm.backward(rows, *[a.at for a in o])  # noqa: E731
        call()
        ha.device.synchronize()
        results.append((operands[5], operands[5].back()))
        calls.append(call)
    at_once(calls)
    assert all(np.array_equal(a.back(), want) for a, want in results)


def test_products_in_shares(gpu, monkeypatch):
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", "4")
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", "4")
    calls, results = [], []
    for k in range(THREADS):   # (of handles of their own, which have the scratch in common)
        op = ha.Int8Matmul(3000, 120 + k, "f32")
        assert "shares=4" in op.describe(130)
        host = int8_inputs(130, 3000, 120 + k, False, seed=k)
        operands = [Array(host[n]) for n in ("x", "x_scales", "weights", "weight_scales")] + [empty((130, 120 + k), np.float32)]
        call = lambda o=operands, op=op: op.multiply(130, *[a.at for a in o])  # noqa: E731
        call()
        ha.device.synchronize()
        results.append((operands[4], operands[4].back()))
        calls.append(call)
    at_once(calls)
    assert all(np.array_equal(a.back(), want) for a, want in results)


def test_clipping(gpu):
    sizes, dtypes = [200_000, 33], ["f32", "bf16"]
    clip = ha.GradientClip(sizes, dtypes)
    calls, results = [], []
    for k in range(THREADS):
        host, _ = clip_inputs(sizes, dtypes, 0.1 * (k + 1), seed=k)
        d, out, norm = [Array(h) for h in host], [empty(h.shape, h.dtype) for h in host], empty((1,), np.float32)
        call = lambda d=d, out=out, norm=norm: clip.clip([a.at for a in d], [a.at for a in out], 0.5, norm.at)  # noqa: E731
        call()
        ha.device.synchronize()
        results += [(a, a.back()) for a in out + [norm]]
        calls.append(call)
    at_once(calls)
    assert all(np.array_equal(a.back(), want) for a, want in results)
