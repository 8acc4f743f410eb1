"""Scratch of two threads that share a stream: buffers of their own (CPU), and right results from calls at the same time with
the pool switched on (GPU)."""

from __future__ import annotations

import threading

import pytest
import torch


def in_threads(count, work):
    """``work(k)`` of every k at the same time; returns the results, raises the first error."""
    results, errors, start = [None] * count, [], threading.Barrier(count)

    def body(k):
        try:
            start.wait(30)
            results[k] = work(k)
        except BaseException as error:  # noqa: BLE001
            errors.append(error)

    threads = [threading.Thread(target=body, args=(k,)) for k in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    if errors:
        raise errors[0]
    return results


def test_threads_never_share_a_pooled_buffer():
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200.cake._runtime import workspace

    package.configure(cake_workspace_pool_bytes=1 << 16)
    gate = threading.Barrier(3)

    def work(_):
        first = workspace.take("linear_recurrence", "states", (64,), torch.float32, "cpu")
        gate.wait(30)  # everybody holds one
        again = workspace.take("linear_recurrence", "states", (32,), torch.float32, "cpu")
        return first.data_ptr(), again.data_ptr()

    got = in_threads(3, work)
    assert len({first for first, _ in got}) == 3
    assert all(first == again for first, again in got)  # a thread's own buffer is used again
    assert workspace.stats()["cpu"]["entries"] == 3
    assert workspace.release("linear_recurrence") == 3 * 256


@pytest.mark.gpu
def test_two_threads_on_one_stream_with_the_pool():
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    package.configure(cake_workspace_pool_bytes=1 << 28)
    gen = torch.Generator(device="cuda").manual_seed(3)
    inputs, want = [], []
    for k in range(2):
        x = torch.randn(1, 4000 + 700 * k, 64, device="cuda", generator=gen).bfloat16()
        g = -0.1 * torch.rand(x.shape, device="cuda", generator=gen)
        inputs.append((x, g))
        want.append(gated_linear_recurrence(x, g, output_final_state=True))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def work(k):
        with torch.cuda.stream(stream), torch.no_grad():
            return [gated_linear_recurrence(*inputs[k], output_final_state=True) for _ in range(60)]

    got = in_threads(2, work)
    torch.cuda.synchronize()
    for k in range(2):
        for y, final in got[k]:
            assert torch.equal(y, want[k][0]) and torch.equal(final, want[k][1]), k
