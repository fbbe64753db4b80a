"""Calls of two host threads on streams of their own, at the same time: layers in two launches and
rows drawn in parts, whose temporaries come from the library's pool, give what they give alone."""
import threading

import numpy as np
import pytest
import torch

from acfun_amd import capi
from oracle import layers

pytestmark = pytest.mark.gpu


class Caller:
    """A layer of many rows and a draw from long ones, on a stream of its own."""

    def __init__(self, gpu, seed):
        rng = np.random.default_rng(seed)
        self.gpu, self.stream = gpu, torch.cuda.Stream()
        M, N, K, C = 200 + seed, 700, 1000, 60000
        self.sizes = M, N, K, C
        with torch.cuda.stream(self.stream):
            self.x = torch.as_tensor(rng.standard_normal((M, K)), dtype=torch.bfloat16).cuda()
            code = rng.integers(-127, 128, (N, K)).astype(np.int8)
            self.w = [torch.as_tensor(v).cuda() for v in layers.q8_tiles(code, np.full(N, 1e-3, np.float32))]
            self.y = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
            self.logits = torch.as_tensor(rng.standard_normal((3, C)) * 2.5, dtype=torch.float32).cuda()
            self.p, self.u = torch.full((3,), 0.9, device="cuda"), torch.as_tensor(rng.random(3), dtype=torch.float32).cuda()
            self.token = torch.zeros(3, dtype=torch.int32, device="cuda")
            self.stream.synchronize()

    def run(self):
        (M, N, K, C), s = self.sizes, self.stream.cuda_stream
        assert self.gpu.acfun_dev_fc_q8(self.x.data_ptr(), 1, M, K, self.w[0].data_ptr(), self.w[1].data_ptr(), None, N,
                                        self.y.data_ptr(), 0, s) == 0, capi.last_error()
        assert self.gpu.acfun_dev_sample(self.logits.data_ptr(), 0, 3, C, C, None, None, self.p.data_ptr(), None,
                                         self.u.data_ptr(), self.token.data_ptr(), None, s) == 0, capi.last_error()

    def results(self):
        self.stream.synchronize()
        return self.y.float().cpu().numpy(), self.token.cpu().numpy()


def test_two_callers(gpu):
    callers = [Caller(gpu, seed) for seed in (1, 2)]
    for c in callers:
        c.run()
    want, wrong = [c.results() for c in callers], []

    def loop(c, w):
        try:
            for _ in range(25):
                with torch.cuda.stream(c.stream):
                    c.y.zero_()
                    c.token.fill_(-7)
                c.run()
                y, token = c.results()
                if not (np.array_equal(y, w[0]) and np.array_equal(token, w[1])):
                    wrong.append(c)
        except Exception as e:                               # (a thread's own would be lost)
            wrong.append(e)
    threads = [threading.Thread(target=loop, args=a) for a in zip(callers, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
