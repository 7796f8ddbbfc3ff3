"""The 4-bit cache's step and the token log probabilities captured into HIP graphs and replayed, on
a stream of the caller's, with eager work between the replays."""
import ctypes as C

import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    N.ensure_init()
    lib = C.CDLL("libamdhip64.so")
    p = C.c_void_p
    lib.hipStreamCreateWithFlags.argtypes = [C.POINTER(p), C.c_uint]
    lib.hipStreamDestroy.argtypes = [p]
    lib.hipStreamSynchronize.argtypes = [p]
    lib.hipStreamBeginCapture.argtypes = [p, C.c_int]
    lib.hipStreamEndCapture.argtypes = [p, C.POINTER(p)]
    lib.hipGraphInstantiate.argtypes = [C.POINTER(p), p, p, p, C.c_size_t]
    lib.hipGraphLaunch.argtypes = [p, p]
    lib.hipGraphExecDestroy.argtypes = [p]
    lib.hipGraphDestroy.argtypes = [p]
    return lib


class Graph:
    """What `work` launches on a stream of its own, captured."""

    def __init__(self, hip, work):
        self.hip, self.stream, own = hip, C.c_void_p(), C.c_void_p()
        assert hip.hipStreamCreateWithFlags(C.byref(self.stream), 1) == 0
        N.check(N.lib.nml_get_stream(C.byref(own)))
        N.synchronize()
        N.check(N.lib.nml_set_stream(self.stream))
        try:
            assert hip.hipStreamBeginCapture(self.stream, 1) == 0
            try:
                work()
            finally:
                graph = C.c_void_p()
                assert hip.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        finally:
            N.check(N.lib.nml_set_stream(own))
        self.exec = C.c_void_p()
        assert hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, 0) == 0
        hip.hipGraphDestroy(graph)

    def run(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def wait(self):
        assert self.hip.hipStreamSynchronize(self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exec)
        self.hip.hipStreamDestroy(self.stream)


def dev(x):
    return N.DeviceArray.from_host(np.ascontiguousarray(x))


def test_replayed_steps_follow_their_inputs(gpu, hip):
    """Two captured steps (write a token, attend), one in pieces and one not, each on a workspace of
    its own, replayed together; positions, keys and queries change between replays."""
    r = np.random.RandomState(0)
    steps = []
    for b, kv, g, dk, p in ((2, 2, 1, 64, 6000), (5, 3, 2, 32, 200)):
        s = {"c": K.KV4Cache(b, kv, p, dk), "shape": (b, kv, g, dk, p)}
        n = p - 40
        k, v = r.randn(b, kv, n, dk).astype(np.float16), r.randn(b, kv, n, dk).astype(np.float16)
        K.kv4_write(s["c"], k, v)
        s["k"], s["v"] = np.zeros((b, kv, p, dk), np.float16), np.zeros((b, kv, p, dk), np.float16)
        s["k"][:, :, :n], s["v"][:, :, :n] = k, v
        s["new"] = [dev(np.zeros((b, kv, 1, dk), np.float16)) for _ in range(2)]
        s["q"] = dev(np.zeros((b, kv * g, 1, dk), np.float16))
        s["pos"], s["lens"] = dev(np.zeros(b, np.int32)), dev(np.ones(b, np.int32))
        s["out"] = dev(np.zeros((b, 1, kv * g * dk), np.float16))
        need = C.c_size_t()
        N.check(N.lib.nml_kv4_attention_workspace(b, kv * g, kv, 1, p, dk, C.byref(need)))
        s["ws"] = dev(np.zeros(max(need.value, 16), np.uint8))

        def work(s=s, b=b, kv=kv, g=g, dk=dk, p=p):
            N.check(N.lib.nml_kv4_write_device(
                s["new"][0].ptr, s["new"][1].ptr, kv * dk, dk, dk, *s["c"].pointers, s["pos"].ptr,
                None, b, kv, 1, p, dk, None, N.F16))
            N.check(N.lib.nml_kv4_attention_device(
                s["q"].ptr, *s["c"].pointers, s["lens"].ptr, None, s["out"].ptr, b, kv * g, kv, 1, p,
                dk, 8.0, s["ws"].ptr, s["ws"].nbytes, None, N.F16))

        s["graph"] = Graph(hip, work)
        steps.append(s)
    for t in range(6):
        want = []
        for s in steps:
            b, kv, g, dk, p = s["shape"]
            pos = r.randint(0, p, b)
            new = [r.randn(b, kv, 1, dk).astype(np.float16) for _ in range(2)]
            q = r.randn(b, kv * g, 1, dk).astype(np.float16)
            for x, y in ((s["new"][0], new[0]), (s["new"][1], new[1]), (s["q"], q),
                         (s["pos"], pos.astype(np.int32)), (s["lens"], (pos + 1).astype(np.int32))):
                N.check(N.lib.nml_memcpy_h2d(x.ptr, y.ctypes.data, y.nbytes))
            for i in range(b):
                s["k"][i, :, pos[i]], s["v"][i, :, pos[i]] = new[0][i, :, 0], new[1][i, :, 0]
            want.append(R.attention(q, R.held(s["k"]), R.held(s["v"]), pos + 1, None, 8.0))
        for s in steps:
            s["graph"].run()
        for s, w in zip(steps, want):
            s["graph"].wait()
            got = s["out"].numpy().astype(np.float64)
            # float16 outputs of values up to 5, probabilities with 17 bits, float32 sums of 6000
            assert np.abs(got - w).max() <= 5 * (2.0**-11 + 2.0**-16 + 6000 * 2.0**-24), t
    # eager calls on the library's stream give the same bits as the replay
    for s in steps:
        b, kv, g, dk, p = s["shape"]
        again = K.kv4_attention(s["q"], s["c"], s["lens"], 8.0).numpy()
        assert np.array_equal(again, s["out"].numpy())
        s["graph"].close()


def test_replayed_log_probabilities(gpu, hip):
    r = np.random.RandomState(1)
    rows, v = 7, 5003
    x, t = dev(np.zeros((rows, v), np.float32)), dev(np.zeros(rows, np.int64))
    stat = [dev(np.zeros(rows, np.float32)) for _ in range(4)]
    ids, top = dev(np.zeros((rows, 6), np.int64)), dev(np.zeros((rows, 6), np.float32))
    dl, d = dev(r.randn(rows).astype(np.float32)), dev(np.zeros((rows, v), np.float32))

    def work():
        N.check(N.lib.nml_token_logprobs_device(
            x.ptr, v, t.ptr, rows, v, 0, 0, 6, stat[0].ptr, stat[1].ptr, stat[2].ptr, stat[3].ptr,
            ids.ptr, top.ptr, None, N.F32))
        N.check(N.lib.nml_token_logprobs_backward_device(
            x.ptr, v, t.ptr, stat[2].ptr, stat[3].ptr, stat[1].ptr, dl.ptr, None, rows, v, 0, 0,
            d.ptr, v, None, N.F32))

    g = Graph(hip, work)
    for _ in range(4):
        logits, targets = (3 * r.randn(rows, v)).astype(np.float32), r.randint(0, v, rows)
        N.check(N.lib.nml_memcpy_h2d(x.ptr, logits.ctypes.data, logits.nbytes))
        N.check(N.lib.nml_memcpy_h2d(t.ptr, targets.ctypes.data, targets.nbytes))
        g.run()
        g.wait()
        eager = [a.numpy() for a in K.token_logprobs(logits, targets, 6)]
        for got, want in zip((stat[0], stat[1], stat[2], stat[3], ids, top), eager):
            assert np.array_equal(got.numpy(), want)
        want = R.logprobs_grad(logits, targets, dl.numpy().astype(np.float64), np.zeros(rows))
        assert np.abs(d.numpy() - want).max() <= 1e-5
    g.close()
