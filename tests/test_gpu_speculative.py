"""The target's side in use: a paged cache through steps, crops and evictions
against a plain one, and speculative generation on small random Qwen2 models."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kvr(built_lib):
    import kv_reduce_b200

    return kv_reduce_b200


def plain_attention(q, ks, vs):
    """q [HQ, T, D] over one sequence's [n, H, D], in 64 bits."""
    HQ, T, D = q.shape
    n, H = ks.shape[:2]
    out = torch.zeros(HQ, T, D, dtype=torch.float64, device=q.device)
    weights = torch.zeros(n, dtype=torch.float64, device=q.device)
    for t in range(T):
        m = n - T + t + 1
        s = torch.einsum("hgd,nhd->hgn", q[:, t].double().view(H, HQ // H, D), ks[:m].double()) * D ** -0.5
        p = torch.softmax(s, -1)
        out[:, t] = torch.einsum("hgn,nhd->hgd", p, vs[:m].double()).reshape(HQ, D)
        weights[:m] += p.sum((0, 1))
    return out, weights


@pytest.mark.parametrize("page", [8, 16, 5])
def test_cache_through_rounds(kvr, page):
    """Ragged acceptance: every round advances all sequences by five tokens and
    crops each to another length; weights and evictions follow."""
    B, HQ, H, D, L = 3, 8, 2, 64, 2
    g = torch.Generator(device="cuda").manual_seed(page)
    cache = kvr.PagedKVCache(L, B, H, D, num_pages=120 // page * B + 40, page_size=page, max_pages=-(-120 // page),
                             track_weights=True)
    keys = [[torch.zeros(0, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(B)] for _ in range(L)]
    values = [[k.clone() for k in row] for row in keys]
    weights = [[torch.zeros(0, dtype=torch.float64, device="cuda") for _ in range(B)] for _ in range(L)]

    def step(T):
        cache.advance(T)
        for layer in range(L):
            k, v, q = (torch.randn(B, T, h, D, device="cuda", generator=g).to(torch.bfloat16).transpose(1, 2)
                       for h in (H, H, HQ))
            cache.append(layer, k, v)
            out = cache.attention(layer, q)
            for b in range(B):
                keys[layer][b] = torch.cat([keys[layer][b], k[b].transpose(0, 1)])
                values[layer][b] = torch.cat([values[layer][b], v[b].transpose(0, 1)])
                want, w = plain_attention(q[b], keys[layer][b], values[layer][b])
                assert (out[b].double() - want).abs().max() < 2 ** -7 * values[layer][b].abs().max()
                weights[layer][b] = torch.cat([weights[layer][b], w.new_zeros(T)]) + w

    def crop(lengths):
        cache.crop(lengths)
        for layer in range(L):
            for b, n in enumerate(lengths):
                keys[layer][b], values[layer][b] = keys[layer][b][:n], values[layer][b][:n]
                weights[layer][b] = weights[layer][b][:n]

    step(30)
    for rnd in range(6):
        held = cache.seq_lengths()
        step(5)
        crop([n + 1 + (rnd * (b + 1) + b) % 5 for b, n in enumerate(held)])
        keep, recent, first = 36, 10, 2
        lengths = cache.seq_lengths()
        if cache.evict(keep, recent=recent, first=first):
            for layer in range(L):
                for b, n in enumerate(lengths):
                    if n <= keep:
                        continue
                    w = weights[layer][b].clone()
                    got = cache.token_weights[layer][b, :keep].double()
                    w[:first] = w[n - recent:] = float("inf")
                    kept = w.topk(keep).indices.sort().values
                    assert torch.allclose(got, weights[layer][b][kept], rtol=1e-4, atol=1e-5)
                    keys[layer][b], values[layer][b] = keys[layer][b][kept], values[layer][b][kept]
                    weights[layer][b] = weights[layer][b][kept]
        for b in range(B):
            n = cache.seq_lengths()[b]
            assert n == len(keys[0][b])
            assert torch.allclose(cache.token_weights[1][b, :n].double(), weights[1][b], rtol=1e-4, atol=1e-5)


def tiny_qwen2(seed, layers=2):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(seed)
    cfg = transformers.Qwen2Config(vocab_size=512, hidden_size=768, intermediate_size=1024, num_hidden_layers=layers,
                                   num_attention_heads=6, num_key_value_heads=2, max_position_embeddings=4096,
                                   attn_implementation="sdpa")
    return transformers.Qwen2ForCausalLM(cfg).to(device="cuda", dtype=torch.bfloat16).eval()


@torch.inference_mode()
def test_target_hook_matches_the_model(built_lib):
    """Several tokens a step over the paged cache: the model's own logits."""
    from kv_reduce_b200 import hf

    model = tiny_qwen2(1)
    ids = torch.randint(0, 512, (1, 130), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want = model(ids).logits.float()
    hf.install_target(model)
    assert torch.equal(model(ids).logits.float(), want)             # other caches are left alone
    cache = hf.PagedTargetCache.for_model(model, 1, max_tokens=160)
    got = [model(ids[:, :100], past_key_values=cache, use_cache=True).logits]
    for a, b in ((100, 101), (101, 106), (106, 130)):
        got.append(model(ids[:, a:b], past_key_values=cache, use_cache=True).logits)
    assert cache.pages.seq_lengths() == [130]
    cos = torch.nn.functional.cosine_similarity(torch.cat(got, 1).float(), want, dim=-1)
    assert cos.min().item() > 0.995
    cache.crop([104])                                               # a rejected tail, then again
    again = model(ids[:, 104:130], past_key_values=cache, use_cache=True).logits.float()
    cos = torch.nn.functional.cosine_similarity(again, want[:, 104:], dim=-1)
    assert cos.min().item() > 0.995


@torch.inference_mode()
def test_greedy_generation_gives_the_targets_tokens(built_lib):
    """Each generated token is the argmax of the target's own forward over the
    tokens before it, up to bf16 noise in the logits."""
    from kv_reduce_b200 import hf

    target, draft = tiny_qwen2(3), tiny_qwen2(3)
    hf.install_target(target)
    hf.install(draft)
    ids = torch.randint(0, 512, (1, 300), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    out, rounds = hf.speculative_generate(target, draft, ids, max_new_tokens=40, draft_tokens=4)
    assert out.shape == (1, 340) and torch.equal(out[:, :300], ids)
    assert sum(rounds) > 0 and len(rounds) < 39                     # the same weights: drafts are accepted
    ref = target(out[:, :-1]).logits[0, 299:].float()
    gap = ref.max(-1).values - ref.gather(1, out[0, 300:, None])[:, 0]
    assert (gap <= 2 ** -5 * ref.abs().max(-1).values).all()


@torch.inference_mode()
@pytest.mark.parametrize("kw", [dict(), dict(window=128, sinks=4), dict(keep=200, recent=64, first=4)])
def test_sampled_generation(built_lib, kw):
    from kv_reduce_b200 import hf

    target, draft = tiny_qwen2(5), tiny_qwen2(5, layers=1)
    hf.install_target(target)
    hf.install(draft)
    ids = torch.randint(0, 512, (1, 260), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    runs = []
    for _ in range(2):
        g = torch.Generator("cuda").manual_seed(7)
        out, rounds = hf.speculative_generate(target, draft, ids, max_new_tokens=24, draft_tokens=3, temperature=0.9,
                                              generator=g, **kw)
        assert out.shape == (1, 284) and 0 <= int(out.min()) and int(out.max()) < 512
        runs.append(out)
    assert torch.equal(*runs)
    with pytest.raises(ValueError):
        hf.speculative_generate(target, draft, ids.expand(2, -1), max_new_tokens=4)
