"""The cache's, the attention's and the drafts' operators as they are used: together, on other streams, captured, by threads; and what they refuse."""
import os
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_generation import Made, ancestors, normal, seeded  # noqa: E402
from verinf_amd.prover import generation as gen  # noqa: E402

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


# ---- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.int8])
def test_a_tree_goes_on_as_if_its_path_had_been_said(kind):
    """Prompts, then trees whose accepted paths are kept: the cache holds what the sequences' tokens put there one after the other, bit for bit, and attention over it
    is what it is over that."""
    dtype = torch.float16 if kind == torch.float16 else torch.bfloat16
    heads, group, dim, page, vocab = 2, 2, 64, 16, 50
    g = seeded(kind.itemsize, dim)
    of_token = {name: normal((vocab, h, dim), g, dtype) for name, h in (("q", heads * group), ("k", heads), ("v", heads))}
    plan = gen.rotary_plan(dim)
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (20, 1, 37)]
    table = torch.randperm(30, generator=g).view(3, 10).int().cuda()
    cache, fresh = gen.new_cache(30, heads, page, dim, kind), gen.new_cache(30, heads, page, dim, kind)

    def say(into, tokens, lengths, positions=None, parents=None):
        """New tokens of each sequence; what they attend to."""
        new = [len(t) for t in tokens]
        starts = torch.tensor([sum(new[:i]) for i in range(4)], dtype=torch.int32).cuda()
        ids = torch.tensor(sum(tokens, []), dtype=torch.long).cuda()
        batch = gen.Batch(starts, torch.tensor(lengths, dtype=torch.int32).cuda(), table)
        at = torch.tensor(positions if positions else sum((list(range(n - k, n)) for n, k in zip(lengths, new)), [])).cuda()
        gen.append_tokens(into, of_token["k"][ids], of_token["v"][ids], batch, at, plan)
        q = gen.rotate_heads(of_token["q"][ids], at, plan)
        return gen.attend_cache(q, into, batch, None if parents is None else torch.tensor(parents, dtype=torch.int32).cuda()), batch, starts, ids

    said = [list(p) for p in prompts]
    lengths = [len(p) - 1 for p in prompts]
    say(cache, [p[:-1] for p in prompts], lengths)
    accepted = 0
    for step in range(4):
        trees, parents, positions = [], [], []
        for b in range(3):
            n = 6 + 3 * b
            parent = [-1] + [int(torch.randint(max(0, (i - 1) // 2), i, (1,), generator=g)) for i in range(1, n)]
            depth = [0] * n
            for i in range(1, n):
                depth[i] = depth[parent[i]] + 1
            trees.append([said[b][-1]] + torch.randint(0, vocab, (n - 1,), generator=g).tolist())
            parents += parent
            positions += [lengths[b] + d for d in depth]
        out, batch, starts, ids = say(cache, trees, [n + len(t) for n, t in zip(lengths, trees)], positions, parents)
        logits = normal((ids.shape[0], vocab), g)
        for i, p in enumerate(parents):        # some drafts are what the target says
            if p >= 0 and i % 3:
                logits[max(x for x in range(i) if parents[x] < 0) + p, ids[i]] += 6.0
        u = torch.rand(ids.shape[0], generator=g, dtype=torch.float64).cuda()
        counts, nodes, tokens = gen.verify_drafts(logits, ids, starts, torch.tensor(parents, dtype=torch.int32).cuda(), u, 5)
        after = gen.keep_drafts(cache, batch, nodes, counts)
        last = []
        for b in range(3):
            k = int(counts[b])
            accepted += k
            path = nodes[b, :k].tolist()
            for d, node in enumerate(path):
                assert trees[b][node] == int(tokens[b, d])
            last.append(path[-1] if path else 0)
            said[b] += tokens[b, :k + 1].tolist()
            lengths[b] += 1 + k
        assert after.tolist() == lengths and all(len(s) == n + 1 for s, n in zip(said, lengths))
        # the same sequences, one token after the other
        for t in (fresh.keys, fresh.values):
            t.zero_()
        alone, *_ = say(fresh, [s[:-1] for s in said], lengths)
        for b in range(3):
            j = torch.arange(lengths[b])
            at, row = table[b, j // page].long(), (j % page).cuda()
            for name in ("keys", "values") + (("key_scales", "value_scales") if kind == torch.int8 else ()):
                assert torch.equal(getattr(cache, name)[at, :, row], getattr(fresh, name)[at, :, row]), (step, b, name)
            end = sum(lengths[:b + 1]) - 1
            # each within a rounding of P and one of the result
            assert ((alone[end].float() - out[int(starts[b]) + last[b]].float()).abs() <= 4 * torch.finfo(dtype).eps * 4).all()
    assert accepted > 0


def test_a_tree_is_each_of_its_paths():
    """Every node attends to what it would as the end of a chain."""
    m = Made(torch.bfloat16, [45], [30], 2, 128, 16)
    parents = [-1] + [(i - 1) // 3 for i in range(1, 30)]
    q = normal((30, 4, 128), seeded(3), torch.bfloat16)
    out = gen.attend_cache(q, m.cache, m.batch, torch.tensor(parents, dtype=torch.int32).cuda())
    seen = ancestors(parents)
    for leaf in (0, 5, 17, 29):
        path = seen[leaf].nonzero()[:, 0].tolist()
        chain = gen.new_cache(8, 2, 16, 128)
        j = list(range(45)) + [45 + i for i in path]
        page, row = (t.cuda() for t in m.places(0, j))
        table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
        to = torch.arange(len(j))
        for name in ("keys", "values"):
            getattr(chain, name)[(to // 16).cuda(), :, (to % 16).cuda()] = getattr(m.cache, name)[page, :, row]
        batch = gen.Batch(torch.tensor([0, len(path)], dtype=torch.int32).cuda(), torch.tensor([len(j)], dtype=torch.int32).cuda(), table)
        alone = gen.attend_cache(q[path], chain, batch)
        assert ((alone.float() - out[path].float()).abs() <= 2 * 2.0 ** -8 * 4).all()          # two roundings each, of values up to 4


def test_the_example_runs(capsys):
    import draft_answer
    model = draft_answer.Model(hidden=256, layers=2, heads=4, shared=2, vocab=300)
    prompts = torch.randint(0, 300, (3, 40), generator=torch.Generator().manual_seed(1)).cuda()
    out, steps = draft_answer.answer(model, prompts, 20, nodes=8)
    assert len(out) == 3 and steps >= 1 and all(0 <= t < 300 for o in out for t in o) and max(len(o) for o in out) >= 20


# ---- streams, graphs, threads -------------------------------------------------------------------------------------
def step_of(m, q, k, v, plan, logits, tokens, u, parents, longest=None):
    gen.append_tokens(m.cache, k, v, m.batch, plan=plan)
    out = gen.attend_cache(gen.rotate_heads(q, torch.arange(q.shape[0], device="cuda"), plan), m.cache, m.batch, parents, longest=longest)
    counts, nodes, said = gen.verify_drafts(logits, tokens, m.batch.starts, parents, u, 4, draft_logits=logits * 0.5)
    return out, counts, nodes, said, gen.keep_drafts(m.cache, m.batch, nodes, counts)


def a_step(seed, before=(900, 40), new=(5, 9)):
    m = Made(torch.bfloat16, list(before), list(new), 2, 64, 16, seed=seed)
    g = seeded(seed, 77)
    n = m.n
    parents = torch.tensor(sum(([-1] + [i // 2 for i in range(x - 1)] for x in new), []), dtype=torch.int32).cuda()
    return m, (normal((n, 8, 64), g, torch.bfloat16), normal((n, 2, 64), g, torch.bfloat16), normal((n, 2, 64), g, torch.bfloat16), gen.rotary_plan(64), normal((n, 3000), g) * 3,
               torch.randint(0, 3000, (n,), generator=g).cuda(), torch.rand(n, generator=g, dtype=torch.float64).cuda(), parents)


def everything(m, results):
    return [t.clone() for t in results] + [m.cache.keys.clone(), m.cache.values.clone()]


def test_on_another_stream():
    m, args = a_step(1)
    want = everything(m, step_of(m, *args))
    m, args = a_step(1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2000000)
        got = everything(m, step_of(m, *args))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed_with_other_lengths():
    """A graph of a step, replayed while lengths, pages and inputs change, with eager work and other graphs between."""
    m, args = a_step(2)
    other, other_args = a_step(3)
    start = (m.cache.keys.clone(), m.cache.values.clone(), m.batch.lengths.clone())
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step_of(m, *args)
        step_of(other, *other_args)
        s.synchronize()
        one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(one, stream=s):
            got = step_of(m, *args)
        with torch.cuda.graph(two, stream=s):
            step_of(other, *other_args)
    for turn, shorter in enumerate((0, 0, 300, 11, 880, 0)):
        def reset():
            m.cache.keys.copy_(start[0])
            m.cache.values.copy_(start[1])
            m.batch.lengths.copy_(start[2] - torch.tensor([shorter, 0], dtype=torch.int32, device="cuda"))
            args[6].copy_(torch.rand(args[6].shape, generator=seeded(turn), dtype=torch.float64))
        reset()
        want = everything(m, step_of(m, *args))
        torch.cuda.synchronize()
        reset()
        two.replay()
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(everything(m, got), want)), turn


def test_threads_on_one_stream_and_on_their_own():
    steps = [a_step(10 + i) for i in range(4)]
    want = [everything(m, step_of(m, *args)) for m, args in steps]
    for shared in (True, False):
        again = [a_step(10 + i) for i in range(4)]
        got, failed = [None] * 4, []
        torch.cuda.synchronize()

        def work(i):
            try:
                with torch.cuda.stream(torch.cuda.default_stream() if shared else torch.cuda.Stream()):
                    m, args = again[i]
                    got[i] = everything(m, step_of(m, *args))
                    torch.cuda.current_stream().synchronize()
            except Exception as e:             # shown below
                failed.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
        assert not failed and all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_the_same_inputs_give_the_same_bits():
    m, args = a_step(5, before=(5000, 40), new=(3, 200))
    want = everything(m, step_of(m, *args))
    for _ in range(3):
        m, args = a_step(5, before=(5000, 40), new=(3, 200))
        assert all(torch.equal(a, b) for a, b in zip(everything(m, step_of(m, *args)), want))


def test_nothing_to_do():
    m = Made(torch.bfloat16, [10], [3], 2, 64, 16)
    none = gen.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros((0, 4), dtype=torch.int32, device="cuda"))
    q = normal((3, 4, 64), seeded(1), torch.bfloat16)
    was = m.cache.keys.clone()
    gen.append_tokens(m.cache, q[:, :2], q[:, 2:], none)
    assert torch.equal(m.cache.keys, was) and (gen.attend_cache(q, m.cache, none) == 0).all()
    gen.append_tokens(m.cache, q[:0, :2], q[:0, 2:], none)
    assert gen.attend_cache(q[:0], m.cache, none).shape == (0, 4, 64) and gen.rotate_heads(q[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), gen.rotary_plan(64)).shape == (0, 4, 64)
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    c, n, o = gen.verify_drafts(normal((3, 9), seeded(1)), empty.new_zeros(3), torch.zeros(1, dtype=torch.int32, device="cuda"), None, torch.zeros(3, dtype=torch.float64, device="cuda"), 2)
    assert c.shape == (0,) and n.shape == (0, 2) and o.shape == (0, 3)
    c, n, o = gen.verify_drafts(normal((0, 9), seeded(1)), empty, torch.zeros(3, dtype=torch.int32, device="cuda"), None, torch.zeros(0, dtype=torch.float64, device="cuda"), 2)
    assert c.tolist() == [0, 0] and (n == -1).all() and (o == -1).all()
    assert gen.keep_drafts(m.cache, none, empty.view(0, 5), empty).shape == (0,)


# ---- refusals -----------------------------------------------------------------------------------------------------
def test_functions_refuse():
    m = Made(torch.bfloat16, [10], [3], 2, 64, 16)
    f = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")         # noqa: E731
    i32, i64 = (lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")), (lambda *s: torch.zeros(s, dtype=torch.int64, device="cuda"))
    plan, u = gen.rotary_plan(64), torch.zeros(3, dtype=torch.float64, device="cuda")
    q, k, logits = f(3, 4, 64), f(3, 2, 64), torch.zeros(3, 9, device="cuda")
    grads, twin = f(3, 4, 64).requires_grad_(), f(3, 64, 4).transpose(1, 2)

    def refused(word, call, *args, **more):
        with pytest.raises(RuntimeError, match=word):
            call(*args, **more)

    refused("dimensions", gen.rotate_heads, f(3, 64), i64(3), plan)
    refused("unit column stride", gen.rotate_heads, twin, i64(3), plan)
    refused("gradient", gen.rotate_heads, grads, i64(3), plan)
    refused("dtype", gen.rotate_heads, i64(3, 4, 64), i64(3), plan)
    refused("dtype", gen.rotate_heads, q, i32(3), plan)
    refused("4 elements", gen.rotate_heads, q, i64(4), plan)
    refused("64 of 32", gen.rotate_heads, f(3, 4, 32), i64(3), plan)
    refused("rotary_plan", gen.rotate_heads, q, i64(3), None)
    refused("on cpu", gen.rotate_heads, q, i64(3), gen.rotary_plan(64, device="cpu"))
    refused("out is", gen.rotate_heads, q, i64(3), plan, out=f(3, 4, 32))
    refused("overlap", gen.rotate_heads, q, i64(3), plan, out=f(3, 1, 64).expand(3, 4, 64))
    refused("heads of 63", gen.rotate_heads, f(3, 4, 63), i64(3), gen.rotary_plan(2))

    refused("dtype", gen.Cache, torch.zeros(4, 2, 16, 64, device="cuda"), f(4, 2, 16, 64))
    refused("values are", gen.Cache, f(4, 2, 16, 64), f(4, 2, 32, 64))
    refused("powers of two", gen.Cache, f(4, 2, 24, 64), f(4, 2, 24, 64))
    refused("powers of two", gen.Cache, f(4, 2, 16, 72), f(4, 2, 16, 72))
    refused("overlap", gen.Cache, f(1, 2, 16, 64).expand(4, 2, 16, 64), f(4, 2, 16, 64))
    refused("multiples of 16 bytes", gen.Cache, f(4, 2, 16, 68)[..., :64], f(4, 2, 16, 64))
    refused("multiples of 16 bytes", gen.Cache, f(4, 2, 16, 80)[..., 1:65], f(4, 2, 16, 64))
    refused("int8", gen.Cache, f(4, 2, 16, 64), f(4, 2, 16, 64), torch.zeros(4, 2, 16, device="cuda"), None)
    refused("Tensor", gen.Cache, f(4, 2, 16, 64).to(torch.int8), f(4, 2, 16, 64).to(torch.int8))
    refused("key_scales", gen.Cache, f(4, 2, 16, 64).to(torch.int8), f(4, 2, 16, 64).to(torch.int8), torch.zeros(4, 2, 8, device="cuda"), torch.zeros(4, 2, 16, device="cuda"))
    refused("gradient", gen.Cache, f(4, 2, 16, 64).requires_grad_(), f(4, 2, 16, 64))

    refused("dtype", gen.Batch, i64(2), i32(1), i32(1, 4))
    refused("starts has 3", gen.Batch, i32(3), i32(1), i32(1, 4))
    refused("lengths has 2", gen.Batch, i32(2), i32(2), i32(1, 4))
    refused("unit column stride", gen.Batch, i32(5), i32(4), i32(4, 4).T)

    refused("k is", gen.append_tokens, m.cache, f(3, 2, 64), f(3, 3, 64), m.batch)
    refused("over a cache of 2 heads", gen.append_tokens, m.cache, f(3, 3, 64), f(3, 3, 64), m.batch)
    refused("dtype", gen.append_tokens, m.cache, k, k.float(), m.batch)
    refused("positions has", gen.append_tokens, m.cache, k, k, m.batch, i64(2), plan)

    refused("dtype", gen.attend_cache, q.float(), m.cache, m.batch)
    refused("dtype", gen.attend_cache, q.half(), m.cache, m.batch)
    refused("3 heads", gen.attend_cache, f(3, 3, 64), m.cache, m.batch)
    refused("of 32", gen.attend_cache, f(3, 4, 32), m.cache, m.batch)
    refused("parents has", gen.attend_cache, q, m.cache, m.batch, i32(2))
    refused("out is", gen.attend_cache, q, m.cache, m.batch, out=f(3, 2, 64))
    refused("scale", gen.attend_cache, q, m.cache, m.batch, scale=0.0)

    refused("depth", gen.verify_drafts, logits, i64(3), i32(2), None, u, 257)
    refused("temperature", gen.verify_drafts, logits, i64(3), i32(2), None, u, 2, temperature=0.0)
    refused("draft_logits are", gen.verify_drafts, logits, i64(3), i32(2), None, u, 2, logits[:, :8])
    refused("dtype", gen.verify_drafts, logits, i64(3), i32(2), None, u, 2, logits.half())
    refused("dtype", gen.verify_drafts, logits, i64(3), i32(2), None, u.float(), 2)
    refused("starts has 0", gen.verify_drafts, logits, i64(3), i32(0), None, u, 2)
    refused("at most", gen.verify_drafts, torch.zeros(1, (1 << 20) + 1, device="cuda"), i64(1), i32(2), None, u[:1], 2)

    refused("nodes must", gen.keep_drafts, m.cache, m.batch, i64(2, 3), i64(1))
    refused("counts has", gen.keep_drafts, m.cache, m.batch, i64(1, 3), i64(2))
    refused("depth", gen.keep_drafts, m.cache, m.batch, i64(1, 257), i64(1))


def test_what_a_call_has_checked_cannot_be_changed():
    """A batch's other lengths would be read from where the first ones lay."""
    m = Made(torch.int8, [10], [3], 2, 64, 16)
    for thing, names in ((m.batch, ("starts", "lengths", "pages")), (m.cache, ("keys", "values", "key_scales", "value_scales")), (gen.rotary_plan(64), ("steps", "rotated"))):
        for name in names:
            with pytest.raises(AttributeError, match="cannot be changed"):
                setattr(thing, name, getattr(thing, name))
            with pytest.raises(AttributeError):
                delattr(thing, name)
    with pytest.raises(RuntimeError, match="steps"):
        gen.RotaryPlan(gen.rotary_plan(32).steps, 64, False, 1.0)
    # what the tensors hold is read anew
    q = normal((3, 4, 64), seeded(1), torch.bfloat16)
    first = gen.attend_cache(q, m.cache, m.batch)
    m.batch.lengths.fill_(5)
    assert not torch.equal(gen.attend_cache(q, m.cache, m.batch), first)
