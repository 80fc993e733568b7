"""Drafted tokens through the model (QUICForCausalLM.verify): what comes back is what greedy decoding gives, whatever is drafted,
and the cache is that of the same text."""

import pytest
import torch

from quic_cu_b200 import model as qmodel

pytestmark = pytest.mark.gpu


def _near(got, tokens, logits, tie=2e-2):
    """Equal up to the first near tie of the oracle (after it the texts are different ones); how many were compared."""
    for i, (g, r) in enumerate(zip(got, tokens)):
        if g != r:
            top = torch.topk(logits[i].float(), 2)
            assert (top.values[0] - top.values[1]).item() < tie and g in top.indices.tolist(), (i, g, r)
            return i
    return min(len(got), len(tokens))


def _draft(right, g, vocab):
    """A tree: the right continuation in one branch, wrong tokens before, beside and behind it."""
    ids, parents, at = [], [], 0
    for t in right:
        for _ in range(int(torch.randint(0, 3, (1,), generator=g))):  # wrong siblings come first
            ids.append((t + 1 + int(torch.randint(0, vocab - 1, (1,), generator=g))) % vocab)
            parents.append(at)
        ids.append(t)
        parents.append(at)
        at = len(ids)
    ids.append(int(torch.randint(0, vocab, (1,), generator=g)))
    parents.append(int(torch.randint(0, len(ids), (1,), generator=g)))
    return ids, parents


@pytest.mark.parametrize("lens,most", [([5], 3), ([1, 40, 17], 4), ([120, 3, 64, 65, 9, 30, 77, 2], 6)])
def test_drafts_give_the_greedy_text(tiny_model, lens, most):
    net, ref, _, _ = tiny_model
    g = torch.Generator().manual_seed(len(lens))
    prompts = [torch.randint(0, 2048, (n,), generator=g) for n in lens]
    want = [ref.greedy(p.tolist(), 24) for p in prompts]
    slots = torch.randperm(len(lens) + 2, generator=g)[:len(lens)].tolist()
    cache = net.new_cache(n_slots=len(lens) + 2, s_max=200)
    first, _ = net.prefill(cache, slots, prompts)
    texts = [[t] for t in first.tolist()]
    calls = 0
    while min(len(t) for t in texts) < 20:
        drafts, parents = [], []
        for i, text in enumerate(texts):  # from the oracle's text, as far as it goes
            right = want[i][0][len(text):len(text) + int(torch.randint(0, most + 1, (1,), generator=g))]
            ids, tree = _draft(right, g, 2048)
            drafts.append(torch.tensor(ids) if i % 2 else ids)
            parents.append(tree)
        before = list(cache.host_len)
        out = net.verify(cache, slots, drafts, parents)
        calls += 1
        for i, (s, new) in enumerate(zip(slots, out)):
            assert len(new) >= 1 and cache.host_len[s] == before[s] + len(new) == lens[i] + len(texts[i]) + len(new) - 1
            texts[i] += new
    assert cache.pos[slots].tolist() == [cache.host_len[s] for s in slots]
    assert cache.tok[slots].tolist() == [t[-1] for t in texts]
    compared = sum(_near(t, w[0], w[1]) for t, w in zip(texts, want))
    assert compared >= 20 * len(lens) // 2 and calls < 20
    # the cache is what a prefill of the same text leaves, up to the roundings to fp16 (34 of 2^-11 / sqrt(3), as for decode steps)
    other = net.new_cache(n_slots=len(lens) + 2, s_max=200)
    net.prefill(other, slots, [torch.cat([p, torch.tensor(t[:-1])]) for p, t in zip(prompts, texts)])
    for s in slots:
        n = cache.host_len[s]
        a, b = cache.kv[0, :, s, :, :n].float(), other.kv[0, :, s, :, :n].float()
        worst = ((a - b).transpose(1, 2).flatten(2).norm(dim=-1) / b.transpose(1, 2).flatten(2).norm(dim=-1)).max().item()
        assert worst < 2 * (34 / 3) ** 0.5 * 2 ** -11, worst


def test_the_second_layers_cache(tiny_model):
    """Linears at a quarter of the scale (no attention near one-hot, no near ties: the text repeats itself): what the second layer
    appends went through the first one's attention over the tree, and was moved by the commit."""
    _, _, state, config = tiny_model
    net = qmodel.from_state_dict({k: v * 0.25 if k.endswith("weight_scale") else v for k, v in state.items()}, config)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 2048, (n,), generator=g) for n in (33, 130, 70)]
    cache, plain, other = (net.new_cache(n_slots=3, s_max=256) for _ in range(3))
    first, _ = net.prefill(cache, [2, 0, 1], prompts)
    net.prefill(plain, [2, 0, 1], prompts)
    steps = net.decode(plain, [2, 0, 1], 9)
    texts = [[t] for t in first.tolist()]
    for right in (3, 5):
        drafts, parents = zip(*[_draft(s[len(t) - 1:len(t) - 1 + right], g, 2048) for s, t in zip(steps, texts)])
        for t, new in zip(texts, net.verify(cache, [2, 0, 1], list(drafts), list(parents))):
            t += new
    for t, f, s in zip(texts, first.tolist(), steps):
        assert len(t) >= 10 and t[:10] == [f] + s
    net.prefill(other, [2, 0, 1], [torch.cat([p, torch.tensor(t[:-1])]) for p, t in zip(prompts, texts)])
    for slot, p, t in zip((2, 0, 1), prompts, texts):
        n = p.numel() + len(t) - 1
        assert cache.host_len[slot] == n
        a, b = cache.kv[1, :, slot, :, :n].float(), other.kv[1, :, slot, :, :n].float()
        worst = ((a - b).transpose(1, 2).flatten(2).norm(dim=-1) / b.transpose(1, 2).flatten(2).norm(dim=-1)).max().item()
        assert worst < 2 * (34 / 3) ** 0.5 * 2 ** -11, worst


def test_verify_and_decode_take_turns(tiny_model):
    net, ref, _, _ = tiny_model
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, 2048, (n,), generator=g) for n in (12, 30)]
    want = [ref.greedy(p.tolist(), 20) for p in prompts]
    cache = net.new_cache(n_slots=2, s_max=128)
    first, _ = net.prefill(cache, [0, 1], prompts)
    texts = [[t] for t in first.tolist()]
    for turn in range(3):
        for i, new in enumerate(net.decode(cache, [0, 1], 2)):
            texts[i] += new
        drafts = [w[0][len(t):len(t) + 2] for w, t in zip(want, texts)]  # chains
        for i, new in enumerate(net.verify(cache, [0, 1], drafts)):
            texts[i] += new
        for i, new in enumerate(net.verify(cache, [0, 1], [[], []])):  # nothing drafted: one step
            assert len(new) == 1
            texts[i] += new
    assert sum(_near(t, w[0], w[1]) for t, w in zip(texts, want)) >= 12


def test_un_quantised_weights():
    from quic_cu_b200.checkpoint import qwen_config_dict, synthetic_dense_checkpoint

    net = qmodel.from_state_dict(synthetic_dense_checkpoint(n_layers=2, vocab=2048, seed=5), qwen_config_dict(2, 2048))
    prompt = torch.arange(40)
    caches = [net.new_cache(n_slots=1, s_max=128) for _ in range(2)]
    for c in caches:
        net.prefill(c, [0], [prompt])
    steps = net.decode(caches[0], [0], 6)[0]
    got = net.verify(caches[1], [0], [steps[:5]])[0]
    n = next((i for i, (a, b) in enumerate(zip(got, steps)) if a != b), len(got))
    assert n == len(got) or n >= 1
    a, b = (c.kv[0, :, 0, :, :40 + n].float().transpose(1, 2).flatten(2) for c in caches)
    assert ((a - b).norm(dim=-1) <= 2 * (34 / 3) ** 0.5 * 2 ** -11 * b.norm(dim=-1)).all()


def test_the_right_branch_is_accepted_whole(tiny_model):
    """Every call keeps all of the branch that greedy decoding takes, and the token after it (linears at a quarter of the scale: no
    near ties)."""
    _, _, state, config = tiny_model
    net = qmodel.from_state_dict({k: v * 0.25 if k.endswith("weight_scale") else v for k, v in state.items()}, config)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, 2048, (n,), generator=g) for n in (33, 130, 70, 5)]
    slots = [3, 0, 2, 1]
    cache, plain = (net.new_cache(n_slots=4, s_max=256) for _ in range(2))
    net.prefill(cache, slots, prompts)
    net.prefill(plain, slots, prompts)
    steps = net.decode(plain, slots, 40)
    done = [0] * 4
    for turn in range(4):
        rights = [int(torch.randint(0, 7, (1,), generator=g)) for _ in slots]
        drafts, parents = zip(*[_draft(s[n:n + right], g, 2048) for s, n, right in zip(steps, done, rights)])
        for i, new in enumerate(net.verify(cache, slots, list(drafts), list(parents))):
            # (the last node is drafted at random and may be right by chance)
            assert rights[i] + 1 <= len(new) <= rights[i] + 2
            assert new == steps[i][done[i]:done[i] + len(new)]
            done[i] += len(new)


def test_a_chain_is_accepted_by_un_quantised_weights():
    """All of it, or up to a near tie of the logits that a prefill of the same text gives."""
    from quic_cu_b200.checkpoint import qwen_config_dict, synthetic_dense_checkpoint

    net = qmodel.from_state_dict(synthetic_dense_checkpoint(n_layers=2, vocab=2048, seed=5), qwen_config_dict(2, 2048))
    for start in (0, 500):
        prompt = torch.arange(start, start + 40)
        caches = [net.new_cache(n_slots=1, s_max=128) for _ in range(3)]
        first = [net.prefill(c, [0], [prompt])[0] for c in caches[:2]][0].cpu()
        steps = net.decode(caches[0], [0], 6)[0]
        got = net.verify(caches[1], [0], [steps[:5]])[0]
        _, logits = net.prefill(caches[2], [0], [torch.cat([prompt, first, torch.tensor(steps[:5])])], all_logits=True)
        compared = _near(got, steps, logits[40:].cpu())
        assert len(got) == (6 if compared == 6 else compared + 1)


def test_refusals(tiny_model):
    net, _, _, _ = tiny_model
    cache = net.new_cache(n_slots=3, s_max=32)
    net.prefill(cache, [0, 1], [torch.arange(5), torch.arange(30)])
    for args, error in ((([0, 0], [[1], [1]]), ValueError), (([0], [[1], [2]]), ValueError), (([7], [[1]]), ValueError),
                        (([], []), RuntimeError), (([2], [[1]]), RuntimeError), (([1], [[1, 2]]), RuntimeError),
                        (([0], [[2048]]), ValueError), (([0], [[-1]]), ValueError), (([0], [[1, 2]], [[0, 2]]), ValueError),
                        (([0], [[1, 2]], [[0]]), ValueError), (([0], [[1, 2]], [[0, -1]]), ValueError)):
        with pytest.raises(error):
            net.verify(cache, *args)
    assert cache.host_len == [5, 30, 0]
    assert len(net.verify(cache, [1, 0], [[3], [1, 2, 3]])) == 2
