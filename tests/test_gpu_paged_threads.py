"""The target's operators from several host threads that share a stream."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kvr(built_lib):
    import kv_reduce_b200

    return kv_reduce_b200


def test_threads_on_one_stream(kvr):
    """Sampled verification is two launches whose counters are not zero in
    between; a split attention or another verification enqueued by a second
    thread must not meet them, nor share their scratch."""
    g = torch.Generator(device="cuda").manual_seed(3)
    B, K, V = 12, 3, 20000

    def verification(seed):
        t = torch.randn(B, K + 1, V, device="cuda", generator=g) * 2
        d = (t[:, :K] + 0.7 * torch.randn(B, K, V, device="cuda", generator=g)).to(torch.bfloat16)
        t = t.to(torch.bfloat16)
        e = torch.empty(B, K, V, device="cuda").exponential_(generator=g)
        tokens = (torch.softmax(d.float(), -1) / e).argmax(-1)
        u = torch.rand(B, K, device="cuda", generator=g)
        noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
        return lambda: kvr.verify_draft_tokens(t, d, tokens, u, noise)

    def attention(tokens):
        page = 32
        n = -(-tokens // page)
        k, v = (torch.randn(n, 2, page, 128, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(1, 12, 1, 128, device="cuda", generator=g).to(torch.bfloat16)
        table = torch.randperm(n, device="cuda", generator=g).to(torch.int32)[None]
        lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
        return lambda: kvr.paged_decode_attention(q, k, v, table, lengths, return_lse=True)

    calls = [verification(0), attention(20000), verification(1), attention(3000)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(calls))

    def loop(i):
        start.wait()
        got = [calls[i]() for _ in range(150)]     # (nothing waits for the GPU in here)
        off = [sum((a != b).sum() for a, b in zip(x, want[i])) for x in got]
        wrong.append(int(torch.stack(off).sum()))

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0] * len(calls)
    for call, w in zip(calls, want):               # and nothing is left behind
        assert all(torch.equal(a, b) for a, b in zip(call(), w))
