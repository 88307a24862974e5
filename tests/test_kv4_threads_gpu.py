"""First calls of two threads at once: on a stream that neither has used, both have to make the scratch."""
import threading

import numpy as np
import pytest
import torch

from kv4_util import dev, dev_i, filled
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


def test_decode_first_calls_of_two_threads_on_a_new_stream():
    import wgkv
    rng = np.random.default_rng(31)
    cases = []
    for lens, Hq, D in ((np.array([[9000, 5000]], np.int32), 8, 128),
                        (rng.integers(1, 900, (24, 8)).astype(np.int32), 8, 64)):
        cache, tbl, _, _ = filled(wgkv, rng, lens, D, 64, 16)
        args = (dev(K4.bf16(rng.standard_normal((lens.shape[0], 1, Hq, D)))), cache, dev_i(lens), dev_i(tbl), D ** -0.5)
        cases.append((args, wgkv.paged_decode_kv4(*args)))
    torch.cuda.synchronize()
    wrong = []

    def work(stream, together, args, want):
        with torch.cuda.stream(stream):
            together.wait()
            got = [wgkv.paged_decode_kv4(*args) for _ in range(4)]
            junk = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(2)]  # takes what was freed
            got += [wgkv.paged_decode_kv4(*args) for _ in range(4)]
            stream.synchronize()
            if not all(torch.equal(g, want) for g in got) or not all((j == 7).all() for j in junk):
                wrong.append(1)

    for _ in range(6):
        stream, together = torch.cuda.Stream(), threading.Barrier(2)
        threads = [threading.Thread(target=work, args=(stream, together, *c)) for c in cases]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong
    wgkv.check_errors()
