"""The operators together, as a serving engine uses them: prompts with rotary positions are appended, rows fork, drafts are tried on
the forks in one call, forks are dropped, pools are compacted; each step against caches that never forked, and the attention against
a plain softmax over the de-quantized view."""
from __future__ import annotations

import itertools

import pytest
import torch

import anna_b200
from anna_b200 import KVCacheConfig, Qwen3DynamicCache, Qwen3PageAllocator
from anna_b200.pools import _PageBook
from anna_b200.prefix_block_cache import PrefixBlockPool

HEADS, KV_HEADS, DIM = 8, 2, 128
ROTARY = dict(theta=1e6, sections=(16, 24, 24), interleaved=True)


def new_cache(batch, mode, *, layers=2, page=16, window=24, allocator=None, bits=4):
    config = KVCacheConfig(num_hidden_layers=layers, cache_block_size=page)
    return Qwen3DynamicCache(config, allocator=allocator or Qwen3PageAllocator(config), batch_size=batch, kv_cache_quantization=mode,
                             kv_cache_quant_bits=bits, kv_cache_residual_len=window)


def states(gen, batch, tokens, heads, dtype=torch.bfloat16):
    return torch.randn(batch, heads, tokens, DIM, generator=gen, device="cuda").to(dtype)


def append(cache, k, v, *, dense=False):
    for layer in range(cache.config.num_hidden_layers):
        out = cache.update(k * (1 + layer), v * (1 - 0.5 * layer), layer, require_dense_cache=dense)
    return out


def views(cache):
    """Dense keys and values of every layer, row by row (rows of different lengths are not padded)."""
    out = []
    for layer in range(cache.config.num_hidden_layers):
        k, v, lengths = cache._gather_layer_cache(layer)
        out.append([(k[b, :, :n].clone(), v[b, :, :n].clone()) for b, n in enumerate(lengths.tolist())])
    return out


def assert_same(a, b):
    for x, y in zip(a, b, strict=True):
        for (k1, v1), (k2, v2) in zip(x, y, strict=True):
            assert torch.equal(k1, k2) and torch.equal(v1, v2)


def pages_in_use(cache):
    allocator = cache.allocator
    return [layer.used_pages() for layer in allocator.layers] + [pool.used_pages() for pool in allocator.turboquant_layers]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
@pytest.mark.parametrize("length", [3, 24, 40, 61, 88])
def test_forks_go_on_like_caches_of_their_own(cuda_device, mode, length):
    gen = torch.Generator(device="cuda").manual_seed(length)
    cache = new_cache(2, mode)
    k, v = states(gen, 2, length, KV_HEADS), states(gen, 2, length, KV_HEADS)
    append(cache, k, v)
    cache.rope_deltas = torch.tensor([[3], [-4]], device="cuda")
    rows = [1, 0, 1, 1]
    fork = cache.fork_rows(rows)
    assert fork.get_seq_lengths().tolist() == [length] * 4 and fork.rope_deltas.flatten().tolist() == [-4, 3, -4, -4]
    before = views(cache)
    assert_same(views(fork), [[layer[r] for r in rows] for layer in before])
    # everybody goes on with tokens of its own: forks first, then the source
    alone = new_cache(4, mode)
    append(alone, k[rows], v[rows])
    for tokens in (1, 2, 19, 1):
        k4, v4 = states(gen, 4, tokens, KV_HEADS), states(gen, 4, tokens, KV_HEADS)
        append(fork, k4, v4)
        append(alone, k4, v4)
        assert_same(views(fork), views(alone))
    assert_same(views(cache), before)
    other = new_cache(2, mode)
    append(other, k, v)
    k2, v2 = states(gen, 2, 30, KV_HEADS), states(gen, 2, 30, KV_HEADS)
    append(cache, k2, v2)
    append(other, k2, v2)
    assert_same(views(cache), views(other))
    assert_same(views(fork), views(alone))
    fork.release()
    assert_same(views(cache), views(other))
    cache.release()
    assert pages_in_use(cache) == [0] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_forks_of_forks_of_clones_and_empty_rows(cuda_device, mode):
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = new_cache(1, mode)
    empty = cache.fork_rows([0, 0])
    assert empty.get_seq_lengths().tolist() == [0, 0]
    k, v = states(gen, 1, 50, KV_HEADS), states(gen, 1, 50, KV_HEADS)
    append(cache, k, v)
    want = views(cache)
    family = [cache.clone()]
    family += [family[0].fork_rows([0]), cache.fork_rows([0, 0])]
    family.append(family[1].fork_rows([0, 0, 0]))
    for member in family:
        for row in range(member.get_batch_size()):
            assert_same([[layer[row]] for layer in views(member)], want)
    for i, member in enumerate(family):
        x = states(gen, member.get_batch_size(), 3 + i, KV_HEADS)
        append(member, x, x)
    assert_same(views(cache), want)
    for member in family:
        got = views(member)
        for row in range(member.get_batch_size()):
            for layer in range(2):
                n = want[layer][0][0].shape[1] - (24 if mode == "turboquant" else 0)
                assert torch.equal(got[layer][row][0][:, :n], want[layer][0][0][:, :n])
        member.release()
    cache.release()
    assert pages_in_use(cache) == [0] * 4
    with pytest.raises(IndexError, match="fork_rows"):
        cache.fork_rows([1])


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_a_fork_that_fails_keeps_no_pages(cuda_device, mode, monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(2)
    cache = new_cache(2, mode)
    append(cache, states(gen, 2, 61, KV_HEADS), states(gen, 2, 61, KV_HEADS))
    before, held = views(cache), pages_in_use(cache)

    def fails(**_):
        raise RuntimeError("no copy")

    with monkeypatch.context() as patch:
        patch.setattr("anna_b200.cache.run_page_copy", fails)
        with pytest.raises(RuntimeError, match="no copy"):
            cache.fork_rows([0, 1, 1])
    assert pages_in_use(cache) == held
    assert_same(views(cache), before)
    cache.fork_rows([1, 0]).release()
    assert pages_in_use(cache) == held


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
@pytest.mark.parametrize("spare", [0, 5])
def test_compaction_keeps_every_row(cuda_device, mode, spare):
    gen = torch.Generator(device="cuda").manual_seed(6)
    allocator = new_cache(0, mode).allocator
    caches = [new_cache(1 + i % 2, mode, allocator=allocator) for i in range(6)]
    for i, cache in enumerate(caches):
        n = 20 + 37 * i
        append(cache, states(gen, cache.get_batch_size(), n, KV_HEADS), states(gen, cache.get_batch_size(), n, KV_HEADS))
    fork = caches[5].fork_rows([0, 1, 0])  # pages with several owners
    for i in (0, 3, 4):
        caches[i].release()
    kept = [caches[1], caches[2], caches[5], fork]
    want = [views(cache) for cache in kept]
    used = pages_in_use(caches[1])
    with pytest.raises(RuntimeError, match="compact"):
        allocator.compact(kept[:-1])
    assert [views(cache) for cache in kept[:1]][0][0][0][0].shape == want[0][0][0][0].shape  # nothing has changed
    for cache, expected in zip(kept, want):
        assert_same(views(cache), expected)
    before = [layer.capacity() for layer in allocator.layers] + [pool.capacity() for pool in allocator.turboquant_layers]
    released = allocator.compact(kept + kept, spare_pages=spare)
    after = [layer.capacity() for layer in allocator.layers] + [pool.capacity() for pool in allocator.turboquant_layers]
    assert released == sum(before) - sum(after) > 0 and pages_in_use(caches[1]) == used
    assert all(a <= u + spare for a, u in zip(after, used) if u)
    if mode == "turboquant":
        assert all(pool.slot_capacity() == sum(cache.get_batch_size() for cache in kept) for pool in allocator.turboquant_layers)
    for cache, expected in zip(kept, want):
        assert_same(views(cache), expected)
    assert allocator.compact(kept, spare_pages=spare) == 0  # there is nothing left to give back
    # and all of them go on: appends, new caches, attention
    newcomer = new_cache(2, mode, allocator=allocator)
    x = states(gen, 2, 70, KV_HEADS)
    append(newcomer, x, x)
    for cache, expected in zip(kept, want):
        x = states(gen, cache.get_batch_size(), 33, KV_HEADS)
        append(cache, x, x)
        got = views(cache)
        for layer, row in itertools.product(range(2), range(cache.get_batch_size())):
            k = expected[layer][row][0]
            n = k.shape[1] - (24 if mode == "turboquant" else 0)
            if n > 0:
                assert torch.equal(got[layer][row][0][:, :n], k[:, :n])
    for cache in [*kept, newcomer]:
        cache.release()
    assert allocator.compact([]) > 0 and allocator.layers[0].capacity() == 0 == allocator.turboquant_layers[0].capacity()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_shared_prompt_blocks_are_found_after_compaction(cuda_device, mode):
    gen = torch.Generator(device="cuda").manual_seed(7)
    prompt = torch.arange(80)[None]
    k, v = states(gen, 1, 80, KV_HEADS), states(gen, 1, 80, KV_HEADS)
    first = new_cache(1, mode)
    filler = new_cache(1, mode, allocator=first.allocator)
    append(filler, states(gen, 1, 100, KV_HEADS), states(gen, 1, 100, KV_HEADS))
    first.set_prompt_token_ids(prompt)
    append(first, k, v)
    filler.release()
    assert first.allocator.compact([first]) > 0
    second = new_cache(1, mode, allocator=first.allocator)
    second.set_prompt_token_ids(prompt)
    append(second, k, v)
    assert_same(views(second), views(first))
    tables = [cache._tables_of(0)[0] for cache in (first, second)]
    shared = len(set(tables[0]) & set(tables[1]))
    assert shared == (5 if mode == "none" else 3)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("share", [True, False])
def test_update_rotary_is_rotary_then_update(cuda_device, mode, given, share):
    gen = torch.Generator(device="cuda").manual_seed(8)
    batch = 1 if share else 3
    allocator = new_cache(0, mode).allocator
    caches = [new_cache(batch, mode), new_cache(batch, mode, allocator=allocator)]
    if share:  # some of the prompt's blocks are another sequence's pages
        donor = new_cache(1, mode, allocator=allocator)
        q, k, v = (states(gen, 1, 40, h) for h in (HEADS, KV_HEADS, KV_HEADS))
        donor.set_prompt_token_ids(torch.arange(40)[None])
        for layer in range(2):
            donor.update_rotary(q, k, v, layer, require_dense_cache=False, **ROTARY)
        caches[1].set_prompt_token_ids(torch.cat((torch.arange(40), torch.arange(900, 930)))[None])
    for cache in caches:
        cache.rope_deltas = torch.arange(batch, device="cuda")[:, None] * -3
    past = 0
    for tokens in (70, 1, 5):
        q2, k2, v2 = (states(gen, batch, tokens, h) for h in (HEADS, KV_HEADS, KV_HEADS))
        if share and past == 0:
            q2[:, :, :40], k2[:, :, :40], v2[:, :, :40] = q, k, v
            for cache in caches:
                cache.rope_deltas = None if not given else cache.rope_deltas
        positions = torch.randint(0, 4000, (3, batch, tokens), generator=gen, device="cuda") if given else None
        if given and share and past == 0:
            positions[..., :40] = torch.arange(40, device="cuda")
        for layer in range(2):
            deltas = caches[0].rope_deltas
            plain = positions if given else (past + torch.arange(tokens, device="cuda"))[None] + (0 if deltas is None else deltas)
            turned, keys = anna_b200.run_multi_axis_rotary(query=q2, key=k2, positions=plain.expand(batch, tokens) if not given else plain,
                                                           **ROTARY)
            caches[0].update(keys, v2, layer, require_dense_cache=False)
            got, dense_k, dense_v, lengths = caches[1].update_rotary(q2, k2, v2, layer, positions=positions, **ROTARY)
            assert torch.equal(got, turned) and lengths.tolist() == [past] * batch
            assert dense_k.shape[2] == past + tokens == dense_v.shape[2]
        past += tokens
        assert_same(views(caches[1]), views(caches[0]))
    with pytest.raises(ValueError, match="update_rotary"):
        caches[0].update_rotary(q2[:, :, :1], k2, v2, 0)


def attention(query, keys, values, tokens):
    """[Hq, T, D] queries, the last positions of [Hkv, L, D] keys and values, in 64 bits."""
    q = query.double().unflatten(0, (KV_HEADS, -1))
    score = q @ keys.double()[:, None].transpose(-1, -2) * DIM ** -0.5
    length = keys.shape[1]
    hidden = torch.arange(length, device="cuda") > (length - tokens + torch.arange(tokens, device="cuda"))[:, None]
    return (torch.softmax(score.masked_fill(hidden, float("-inf")), dim=-1) @ values.double()[:, None]).flatten(0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 24])
def test_a_request_with_images_drafts_and_candidates(cuda_device, dtype, page):
    """Prompt, fork, drafts on the fork in one call, the accepted ones on the source, compaction in between."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    cache = new_cache(2, "turboquant", page=page, window=32)
    x = {h: states(gen, 2, 300, h, dtype) for h in (HEADS, KV_HEADS)}
    value = states(gen, 2, 300, KV_HEADS, dtype)
    positions = torch.randint(0, 300, (3, 2, 300), generator=gen, device="cuda")
    for layer in range(2):
        cache.update_rotary(x[HEADS], x[KV_HEADS], value, layer, positions=positions, require_dense_cache=False, **ROTARY)
    cache.rope_deltas = torch.tensor([[-50], [-90]], device="cuda")
    # at 4 bits the dense view rounds keys to the cache's type, which the decode does not: half a step of |k| <= 25 on scores of up to
    # |q| |k| / sqrt(D), and the same of the values (|v| <= 6), on top of what the decode's own tests bound
    eps = torch.finfo(dtype).eps
    tol = max(40 * eps, 2e-3)
    for step, tokens in enumerate((4, 1, 7, 2, 12)):
        drafts = cache.fork_rows([0, 1])
        q, k, v = (states(gen, 2, tokens, h, dtype) for h in (HEADS, KV_HEADS, KV_HEADS))
        for layer in range(2):
            turned, keys, values, _ = drafts.update_rotary(q, k, v, layer, **ROTARY)
            got = drafts.turboquant_multi_token_decode_attention(layer, turned, scaling=DIM ** -0.5, num_key_value_groups=HEADS // KV_HEADS)
            for b in range(2):
                want = attention(turned[b], keys[b], values[b], tokens)
                torch.testing.assert_close(got[b].double(), want, atol=tol, rtol=tol)
        before = views(cache)
        drafts.release()
        accepted = tokens // 2 + 1 if tokens > 1 else 1
        for layer in range(2):
            turned, *_ = cache.update_rotary(q[:, :, :accepted], k[:, :, :accepted], v[:, :, :accepted], layer, require_dense_cache=False,
                                             **ROTARY)
            again = cache.turboquant_multi_token_decode_attention(layer, turned, scaling=DIM ** -0.5,
                                                                  num_key_value_groups=HEADS // KV_HEADS)
            assert again.shape == (2, HEADS, accepted, DIM)
        after = views(cache)
        n = before[0][0][0].shape[1] - 32
        assert torch.equal(after[0][0][0][:, :n], before[0][0][0][:, :n])
        if step % 2:
            cache.allocator.compact([cache])
            assert_same(views(cache), after)
    cache.release()
    assert pages_in_use(cache) == [0] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["none", "turboquant"])
def test_a_refused_append_leaves_the_cache_alone(cuda_device, mode):
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache = new_cache(2, mode)
    append(cache, states(gen, 2, 31, KV_HEADS), states(gen, 2, 31, KV_HEADS))
    before, held = views(cache), pages_in_use(cache)
    q, k = states(gen, 2, 5, HEADS), states(gen, 2, 5, KV_HEADS)
    positions = torch.zeros(3, 2, 5, dtype=torch.long, device="cuda")
    for bad in (dict(positions=positions[:, :, :4]), dict(positions=positions.int()), dict(positions=positions[:2]),
                dict(rotary_dim=DIM + 2), dict(rotary_dim=31, sections=None), dict(sections=(1, 2, 3)), dict(theta=-1.0),
                dict(positions=positions.cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            cache.update_rotary(q, k, k, 0, **{**ROTARY, **bad})
    for k2 in (k[:, :1], k[..., :64], k.float()):
        q2 = q[..., :k2.shape[-1]].to(k2.dtype)
        with pytest.raises((RuntimeError, ValueError)):
            cache.update_rotary(q2, k2, k2, 0)
    with pytest.raises((RuntimeError, ValueError)):
        cache.update_rotary(q, k, k.half(), 0, **ROTARY)
    assert cache.layer_lengths == [[31, 31], [31, 31]] and pages_in_use(cache) == held
    assert_same(views(cache), before)
    cache.update_rotary(q, k, k, 0, **ROTARY)
    assert cache.layer_lengths[0] == [36, 36]


@pytest.mark.gpu
def test_a_compaction_that_runs_out_of_memory_keeps_every_row(cuda_device, monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(6)
    allocator = Qwen3PageAllocator(KVCacheConfig(num_hidden_layers=2, cache_block_size=16))
    caches = [new_cache(2, mode, allocator=allocator) for mode in ("none", "turboquant", "none", "turboquant")]
    for cache in caches:
        append(cache, states(gen, 2, 77, KV_HEADS), states(gen, 2, 77, KV_HEADS))
    for cache in caches[:2]:
        cache.release()
    caches = caches[2:]
    before, gather = [views(cache) for cache in caches], anna_b200.page_copy.run_page_gather
    for works in range(6):  # two layers, each with un-quantized pages, packed pages and rings
        left = [works]

        def some(**arguments):
            if left[0] == 0:
                raise torch.cuda.OutOfMemoryError("no room")
            left[0] -= 1
            return gather(**arguments)

        with monkeypatch.context() as patch:
            patch.setattr("anna_b200.page_copy.run_page_gather", some)
            try:
                allocator.compact(caches)
            except torch.cuda.OutOfMemoryError:
                pass
        for cache, want in zip(caches, before):
            assert_same(views(cache), want)
    for cache in caches:
        append(cache, states(gen, 2, 40, KV_HEADS), states(gen, 2, 40, KV_HEADS))
    for cache, want in zip(caches, before):
        for new, old in zip(views(cache), want, strict=True):
            for (k, v), (k0, v0) in zip(new, old, strict=True):
                if cache.kv_cache_quantization == "none":
                    assert torch.equal(k[:, :77], k0) and torch.equal(v[:, :77], v0)


@pytest.mark.gpu
def test_multi_token_attention_of_the_cache(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(10)
    cache = new_cache(3, "turboquant", layers=1)
    q = states(gen, 3, 4, HEADS)
    call = dict(scaling=DIM ** -0.5, num_key_value_groups=HEADS // KV_HEADS)
    assert torch.count_nonzero(cache.turboquant_multi_token_decode_attention(0, q, **call)) == 0  # nothing appended yet
    x = states(gen, 3, 2, KV_HEADS)
    cache.update(x, x, 0, require_dense_cache=False)  # no packed page, fewer tokens than queries
    got = cache.turboquant_multi_token_decode_attention(0, q, **call)
    assert torch.count_nonzero(got[:, :, :2]) == 0 and bool((got[:, :, 2:].abs().sum(-1) > 0).all())
    torch.testing.assert_close(got[:, :, 2], x[:, :, 0].repeat_interleave(4, dim=1), atol=0, rtol=2 ** -8)  # one key: its value
    x = states(gen, 3, 90, KV_HEADS)
    cache.update(x, x, 0, require_dense_cache=False)
    together = cache.turboquant_multi_token_decode_attention(0, q, **call)
    single = cache.turboquant_single_token_decode_attention(0, q[:, :, 3:], **call)
    torch.testing.assert_close(together[:, :, 3:], single, atol=2e-2, rtol=2e-2)
    # rows of several lengths, stacked, before anything was appended to the batch
    caches = []
    for n in (30, 200, 5):
        part = new_cache(1, "turboquant", layers=1, allocator=cache.allocator)
        y = states(gen, 1, n, KV_HEADS)
        part.update(y, y, 0, require_dense_cache=False)
        caches.append(part)
    each = [part.turboquant_multi_token_decode_attention(0, q[:1], **call) for part in caches]
    stacked = Qwen3DynamicCache.stack(caches, cache.config, clone_turboquant_rows=False)
    got = stacked.turboquant_multi_token_decode_attention(0, q[:1].expand(3, -1, -1, -1), **call)
    torch.testing.assert_close(got, torch.cat(each), atol=1e-2, rtol=1e-2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = stacked.turboquant_multi_token_decode_attention(0, q[:1].expand(3, -1, -1, -1), **call)
    side.synchronize()
    assert torch.equal(again, got)
    for bad, match in ((dict(query_states=q[0]), "query_states"), (dict(query_states=q[:2]), "batch size"), (dict(gate=q[:, :, :1]), "gate"),
                       (dict(num_key_value_groups=2), "query heads"), (dict(query_states=q[..., :64]), "head_dim"),
                       (dict(query_states=q.half()), "dtype")):
        error = RuntimeError if match == "dtype" else ValueError
        with pytest.raises(error, match=match):
            cache.turboquant_multi_token_decode_attention(**{**dict(layer_idx=0, query_states=q, **call), **bad})


def test_books_are_renumbered():
    book = _PageBook()
    ids, _, _ = book.take(10, 16)
    book.retain(ids[3])
    book.release_many([ids[0], ids[5]])
    live = {page: new for new, page in enumerate(sorted(book.refcount))}
    book.renumber(live, len(live) + 2)
    assert book.refcount == {new: 2 if old == ids[3] else 1 for old, new in live.items()}
    assert book.free_pages == [9, 8] and book.take(1, 10)[0] == [8]


def test_registered_blocks_move_with_their_pages():
    pool = PrefixBlockPool()
    pool.register(0, (1, 2), 7)
    pool.register(0, (3, 4), 9)
    pool.register(1, (1, 2), 7)
    pool.move_pages(0, {7: 0, 5: 1})
    assert pool.lookup(0, (1, 2)) == 0 and pool.lookup(0, (3, 4)) is None and pool.lookup(1, (1, 2)) == 7
    pool.discard_page(0, 7)
    assert pool.lookup(0, (1, 2)) == 0
    pool.discard_page(0, 0)
    assert pool.lookup(0, (1, 2)) is None and len(pool) == 1


def test_compaction_refuses_what_it_cannot_do():
    a, b = new_cache(1, "none"), new_cache(1, "none")
    with pytest.raises(ValueError, match="another allocator"):
        a.allocator.compact([a, b])
    with pytest.raises(ValueError, match="spare_pages"):
        a.allocator.compact([a], spare_pages=-1)
    assert a.allocator.compact([a]) == 0
    a.allocator.layers[1]._book.take(1, 16)  # a page that no cache maps
    with pytest.raises(RuntimeError, match="layer 1 has 1 owners"):
        a.allocator.compact([a])
    with pytest.raises(IndexError, match="fork_rows"):
        a.fork_rows([-1])
    with pytest.raises(RuntimeError, match="CUDA"):
        a.update_rotary(torch.zeros(1, 8, 2, 128), torch.zeros(1, 2, 2, 128), torch.zeros(1, 2, 2, 128), 0)
    with pytest.raises(ValueError, match="TurboQuant"):
        a.turboquant_multi_token_decode_attention(0, torch.zeros(1, 8, 2, 128), scaling=1.0, num_key_value_groups=4)
