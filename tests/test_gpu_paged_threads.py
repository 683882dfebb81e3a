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


def test_decode_threads_whose_scratch_grows(kvr):
    """Packed decodes of rising sizes beside small ones, on one stream: a call's
    buffers are its own until it is launched, though another outgrows them."""
    g = torch.Generator(device="cuda").manual_seed(4)
    calls = []
    for B, S in ((1, 600), (2, 3000), (8, 3000), (16, 6000), (24, 9000)):
        k, v = (torch.randn(B, 2, S, 128, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(B, 12, 1, 128, device="cuda", generator=g).to(torch.bfloat16)
        pk, pv = kvr.pack_kivi_kv(k, v, k_bits=4, v_bits=4, group_size=32, residual_length=128)
        calls.append(lambda q=q, pk=pk, pv=pv: kvr.packed_kv_decode_attention(q, pk, pv))
    s = torch.cuda.Stream()                        # (a stream of its own: nothing has grown its scratch yet)
    s.wait_stream(torch.cuda.current_stream())
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(3)

    def loop(order):
        start.wait()
        with torch.cuda.stream(s):
            got = [(i, calls[i]()) for i in order]
            wrong.append(int(torch.stack([(x != want[i]).sum() for i, x in got]).sum()))

    threads = [threading.Thread(target=loop, args=(o,)) for o in ([0] * 200, [0, 1] * 100,
                                                                 [0] * 40 + [1] * 40 + [2] * 40 + [3] * 40 + [4] * 40)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0] * 3
