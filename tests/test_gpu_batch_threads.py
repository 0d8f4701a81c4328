"""The batch operators called by two threads at once, on streams of their own, with plans that both use."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_two_threads(dev):
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(1)
    counts, of = [1, 40, 1, 7], [1, 0, -1, 1]
    a, b = (torch.randn(2, 16, 256, generator=g) / 16).half().to(dev), (torch.randn(2, 128, 16, generator=g) / 4).half().to(dev)
    plan = ops.adapter_plan(of, counts, 2, dev)
    pages = ops.paged_plan(torch.tensor([[1, 0]], dtype=torch.int32), [70], [0], [49], 4, 2, 64, 64, dev)
    cos, sin = torch.rand(49, 64, generator=g).to(dev), torch.rand(49, 64, generator=g).to(dev)
    index = torch.tensor([2, 2, 0, 3], device=dev)
    inputs = []
    for _ in range(2):
        inputs.append({"x": torch.randn(49, 256, generator=g).half().to(dev), "base": torch.randn(49, 128, generator=g).half().to(dev),
                       "qkv": torch.randn(49, 8, 64, generator=g).half().to(dev), "logits": torch.randn(3, 4, 5000, generator=g).to(dev),
                       "scores": torch.randn(3, 4, generator=g).to(dev), "state": torch.randn(4, 3, 777, generator=g).to(dev)})

    def calls(s):
        rows, state = torch.zeros(2, 2, 2, 64, 64, dtype=torch.float16, device=dev), s["state"].clone()
        out = [ops.add_adapters(s["base"], s["x"], a, b, plan), ops.paged_rope_append(s["qkv"], cos, sin, rows, pages), rows]
        out += ops.beam_select(s["logits"], s["scores"], stay=True)
        ops.reorder_rows([state], index)
        return out + [state]

    want = [calls(s) for s in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = calls(inputs[i])
                    if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # (an assertion of a thread is nobody's)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
