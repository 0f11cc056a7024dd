"""The attention block (rotation with norms and cache store, paged decode, prompts) against the definitions in 64 bits, at the
sizes, layouts and masks where it can go wrong."""

import pytest
import torch

from oracle import attention as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAN = float("nan")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _close(got, want, bound, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape
    if not got.numel():
        return
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    wrong = (got - want).abs() - bound
    wrong[torch.isnan(want)] = -1
    assert wrong.max().item() <= 0, (what, wrong.max().item(), (got - want).abs().nan_to_num().max().item())


# ---- rotation --------------------------------------------------------------------------------------------------------


def _rotation(t, heads, kv_heads, dim, dtype, seed, packed=True):
    g = _gen(seed)
    qkv = torch.randn(t, (heads + 2 * kv_heads) * dim, generator=g).to(dtype).cuda()
    q, k, v = (p.view(t, -1, dim) for p in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    weights = [(1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2)]
    return q, k, v, weights, g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (128, 64), (64, 0), (8, 0), (16, 16), (24, 16), (96, 96), (80, 32), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_every_head_size(dtype, dim, rotary, interleaved):
    from nanovllm_voxcpm_amd.attention_ops import rotate_qk

    print(dtype, dim, rotary, interleaved, flush=True)
    t, heads, kv_heads, reach = 13, 6, 2, 50
    q, k, v, weights, g = _rotation(t, heads, kv_heads, dim, dtype, 1)
    positions = torch.randint(0, reach, (t,), generator=g)
    table = torch.randn(reach, max(rotary, 1), generator=g)[:, :rotary]
    for norms in (False, True):
        w = weights if norms else [None, None]
        got_q, got_k = rotate_qk(q, k, positions.cuda(), table.cuda(), q_weight=w[0], k_weight=w[1], interleaved=interleaved)
        for got, x, weight in ((got_q, q, w[0]), (got_k, k, w[1])):
            want, bound = oracle.rotate(x.cpu(), positions, table, None if weight is None else weight.cpu(), interleaved=interleaved)
            _close(got, want, bound + want.abs() * oracle.HALF_STEP[dtype] * (1 + 2**-7) + 2.0**-25 * (dtype == torch.float16), (norms, "q" if x is q else "k"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,heads,kv_heads", [(1, 16, 2), (3, 1, 1), (67, 32, 8), (300, 4, 4), (1500, 7, 1)])
def test_rotation_stores_keys_and_values(dtype, t, heads, kv_heads):
    """Rows with a slot are stored, and nothing else of the cache changes: padding, slots behind the last block, other rows."""
    from nanovllm_voxcpm_amd.attention_ops import rotary_table, rotate_qk

    print(dtype, t, heads, kv_heads, flush=True)
    dim, page = 64, 16
    q, k, v, weights, g = _rotation(t, heads, kv_heads, dim, dtype, 2)
    blocks = -(-t // page) + 2
    caches = [torch.randn(blocks, page, kv_heads, dim, generator=g).to(dtype) for _ in range(2)]
    slots = torch.randperm(blocks * page, generator=g)[:t].to(torch.int32)
    if t > 2:
        slots[1], slots[-1] = -1, blocks * page  # padding; behind the last block
    positions = torch.randint(0, 900, (t,), generator=g, dtype=torch.int32)
    table = rotary_table(dim, 900)
    k_cache, v_cache = (c.cuda() for c in caches)
    for slot_type in (torch.int32, torch.int64):
        got_q, none = rotate_qk(q, k, positions.cuda(), table.cuda(), q_weight=weights[0], k_weight=weights[1].float().to(weights[0].dtype), v=v,
                                k_cache=k_cache, v_cache=v_cache, slot_mapping=slots.to(slot_type).cuda())
        assert none is None
    plain_q, plain_k = rotate_qk(q, k, positions.cuda(), table.cuda(), q_weight=weights[0], k_weight=weights[1])
    assert torch.equal(got_q, plain_q)
    want_k, want_v = (c.clone().view(-1, kv_heads, dim) for c in caches)
    kept = (slots >= 0) & (slots < blocks * page)
    want_k[slots[kept].long()], want_v[slots[kept].long()] = plain_k.cpu()[kept], v.cpu()[kept]
    assert torch.equal(k_cache.cpu().view(-1, kv_heads, dim), want_k)
    assert torch.equal(v_cache.cpu().view(-1, kv_heads, dim), want_v)


def test_rotation_in_place_with_other_strides_and_off_alignment():
    from nanovllm_voxcpm_amd.attention_ops import rotary_table, rotate_qk

    t, heads, kv_heads, dim = 29, 4, 2, 64
    table = rotary_table(dim, 64).cuda()
    for dtype in DTYPES:
        q, k, v, weights, g = _rotation(t, heads, kv_heads, dim, dtype, 3)
        positions = torch.randint(0, 64, (t,), generator=g).cuda()
        want = rotate_qk(q, k, positions, table, q_weight=weights[0].float(), k_weight=weights[1].float())
        # heads outside rows; rows at an odd element
        turned_q, turned_k = q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1)
        odd_q = torch.empty(t * heads * dim + 1, dtype=dtype, device="cuda")[1:].view(t, heads, dim).copy_(q)
        for a, b in ((turned_q, turned_k), (odd_q, turned_k)):
            got = rotate_qk(a, b, positions, table, q_weight=weights[0].float(), k_weight=weights[1].float())
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        # in place, in the packed rows
        got = rotate_qk(q, k, positions, table, q_weight=weights[0].float(), k_weight=weights[1].float(), q_out=q, k_out=k)
        assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("t,heads,kv_heads", [(5, 1, 0), (5, 0, 2), (70000, 2, 0), (9001, 5, 3)])
def test_rotation_of_query_heads_or_key_heads_alone_and_of_many_tokens(t, heads, kv_heads):
    from nanovllm_voxcpm_amd.attention_ops import rotary_table, rotate_qk

    g = _gen(20)
    q, k = (torch.randn(t, h, 64, generator=g).to(torch.float16) for h in (heads, kv_heads))
    positions, table = torch.randint(0, 500, (t,), generator=g), rotary_table(64, 500)
    got_q, got_k = rotate_qk(q.cuda(), k.cuda(), positions.cuda(), table.cuda())
    some = torch.randperm(t, generator=g)[:40].sort().values
    for got, x in ((got_q, q), (got_k, k)):
        want, bound = oracle.rotate(x[some], positions[some], table)
        _close(got[some.cuda()], want, bound + want.abs() * 2.0**-11 * (1 + 2**-7) + 2.0**-25)


def test_rotation_by_a_position_outside_the_table_is_nan_and_far_positions_are_right():
    from nanovllm_voxcpm_amd.attention_ops import rotary_table, rotate_qk

    q, k, v, _, g = _rotation(4, 2, 1, 64, torch.float32, 4)
    table = rotary_table(32, 1 << 17)
    positions = torch.tensor([0, (1 << 17) - 1, 1 << 17, -1])
    got, _ = rotate_qk(q, k, positions.cuda(), table.cuda())
    want, bound = oracle.rotate(q.cpu(), positions, table)
    _close(got, want, bound + want.abs() * 2.0**-24)
    assert torch.isnan(got[2:, :, :32]).all() and torch.equal(got[2:, :, 32:], q[2:, :, 32:])
    angle = torch.tensor((1 << 17) - 1, dtype=torch.float64) * 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert (table[-1].double() - torch.cat([angle.cos(), angle.sin()])).abs().max() <= 2.0**-24


# ---- decode ----------------------------------------------------------------------------------------------------------


def _paged(lens, kv_heads, dim, page, dtype, g, spare=2, value=None):
    """Keys and values of every sequence, the same in pages in random order, and the table; unused rows hold NaN."""
    counts = [-(-n // page) for n in lens]
    blocks = sum(counts) + spare
    order = torch.randperm(blocks, generator=g).to(torch.int32)
    caches = [torch.full((blocks, page, kv_heads, dim), NAN, dtype=dtype) for _ in range(2)]
    table = torch.full((len(lens), max(counts + [1]) + 1), -1, dtype=torch.int32)
    dense, at = [], 0
    for s, n in enumerate(lens):
        table[s, : counts[s]] = order[at : at + counts[s]]
        at += counts[s]
        pair = []
        for c in caches:
            x = torch.randn(n, kv_heads, dim, generator=g).to(dtype)
            for j in range(counts[s]):
                part = x[j * page : (j + 1) * page]
                c[table[s, j], : part.size(0)] = part
            pair.append(x)
        dense.append(pair)
    return dense, caches[0].cuda(), caches[1].cuda(), table


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 511, 513]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(16, 2, 64, 16), (8, 8, 128, 64), (32, 8, 128, 16), (7, 1, 64, 256), (32, 1, 64, 32), (6, 2, 96, 16),
                                                     (4, 2, 64, 7), (24, 1, 128, 48), (2, 1, 256, 16), (3, 1, 8, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (70, 4), (16, 100), (500, 1)])
def test_decode_of_every_length(dtype, heads, kv_heads, dim, page, window, sinks):
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    print(dtype, heads, kv_heads, dim, page, window, sinks, flush=True)
    g = _gen(5)
    dense, k, v, table = _paged(LENS, kv_heads, dim, page, dtype, g)
    q = (1.5 * torch.randn(len(LENS), heads, dim, generator=g)).to(dtype)
    got = decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor(LENS, dtype=torch.int32, device="cuda"), window=window, sinks=sinks)
    for s, (kk, vv) in enumerate(dense):
        want, bound = oracle.attend(q[s : s + 1], kk, vv, True, window, sinks, dtype=dtype)
        _close(got[s : s + 1], want, bound, LENS[s])


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 64), (4, 4, 128), (20, 1, 128)])
@pytest.mark.parametrize("sequences", [1, 3])
def test_decode_of_few_long_sequences(heads, kv_heads, dim, sequences):
    """Work is split over the length: parts that end anywhere, one sequence much longer than the others."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    print(heads, kv_heads, dim, sequences, flush=True)
    g = _gen(6)
    lens = [20011, 1, 4097][:sequences]
    for dtype, window, sinks in ((torch.bfloat16, 0, 0), (torch.float16, 9999, 77), (torch.float32, 0, 0)):
        dense, k, v, table = _paged(lens, kv_heads, dim, 64, dtype, g)
        q = (1.5 * torch.randn(sequences, heads, dim, generator=g)).to(dtype)
        args = (q.cuda(), k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
        got = decode_attention(*args, window=window, sinks=sinks)
        for s, (kk, vv) in enumerate(dense):
            want, bound = oracle.attend(q[s : s + 1], kk, vv, True, window, sinks, dtype=dtype)
            _close(got[s : s + 1], want, bound, (dtype, lens[s]))
        assert torch.equal(decode_attention(*args, window=window, sinks=sinks), got)  # (no order of additions depends on timing)


def test_decode_with_scores_far_apart():
    """Maxima that grow by hundreds from key to key, large negative scores, infinite scores."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    g = _gen(7)
    for dtype in DTYPES:
        lens = [300, 300, 300, 70]
        dense, k, v, table = _paged(lens, 1, 64, 16, dtype, g)
        ramp = torch.linspace(-40, 40, 300).to(dtype)
        for s, sign in ((0, 1.0), (1, -1.0)):
            dense[s][0][:, 0, :] = (sign * ramp)[:, None]
        dense[2][0][:, 0, :] = -50.0
        dense[3][0][33, 0, 5] = float("inf")
        for s in range(4):
            for j in range(-(-lens[s] // 16)):
                part = dense[s][0][16 * j : 16 * j + 16]
                k[table[s, j], : part.size(0)] = part.cuda()
        q = torch.ones(4, 2, 64, dtype=dtype) * 3
        q[3, 1, 5] = -1.0
        got = decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=1.0)
        for s in range(3):
            want, bound = oracle.attend(q[s : s + 1], *dense[s], scale=1.0, dtype=dtype)
            _close(got[s : s + 1], want, bound, (dtype, s))
        # a score of +inf leaves NaN, one of -inf a weight of nothing, as a softmax has it
        assert torch.isnan(got[3, 0]).all()
        want, bound = oracle.attend(q[3:, 1:], *dense[3], scale=1.0, dtype=dtype, hidden=(33,))
        terms_without = bound  # (the hidden key's terms are not finite)
        _close(got[3:, 1:], want, terms_without, (dtype, 3))


def test_decode_leaves_pages_outside_the_cache_unread():
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    g = _gen(8)
    for dtype, dim in ((torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.bfloat16, 96)):
        lens = [100, 100, 20]
        dense, k, v, table = _paged(lens, 2, dim, 16, dtype, g)
        table[0, 2], table[1, 0], table[1, 6] = -5, k.size(0), 1 << 30
        table[2, :2] = -1
        q = torch.randn(3, 4, dim, generator=g).to(dtype)
        got = decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
        for s, hidden in ((0, range(32, 48)), (1, [*range(16), *range(96, 100)]), (2, range(20))):
            want, bound = oracle.attend(q[s : s + 1], *dense[s], dtype=dtype, hidden=set(hidden))
            _close(got[s : s + 1], want, bound, (dtype, s))


def test_decode_clamps_lengths_to_the_table():
    from nanovllm_voxcpm_amd.attention_ops import decode_attention

    g = _gen(9)
    dense, k, v, table = _paged([64, 64], 1, 64, 16, torch.bfloat16, g)
    q = torch.randn(2, 1, 64, generator=g).to(torch.bfloat16)
    got = decode_attention(q.cuda(), k, v, table[:, :4].cuda(), torch.tensor([1 << 30, -7], dtype=torch.int32, device="cuda"))
    want, bound = oracle.attend(q[:1], *dense[0], dtype=torch.bfloat16)
    _close(got[:1], want, bound)
    assert not got[1].any()


def test_decode_behind_the_first_4_gb_of_a_cache():
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, rotate_qk

    page, kv_heads, dim = 256, 8, 128
    blocks = (5 << 30) // (page * kv_heads * dim * 2)
    k, v = (torch.zeros(blocks, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = _gen(10)
    n = 300
    kk, vv = (torch.randn(n, kv_heads, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[blocks - 1, blocks - 3]], dtype=torch.int32)
    slots = torch.tensor([int(table[0, j // page]) * page + j % page for j in range(n)])
    q = torch.randn(n, 8, dim, generator=g).to(torch.bfloat16)
    still = torch.zeros(1, 0, dtype=torch.float32, device="cuda")
    rotate_qk(q.cuda(), kk.cuda(), torch.zeros(n, dtype=torch.int64, device="cuda"), still, v=vv.cuda(), k_cache=k, v_cache=v, slot_mapping=slots.cuda())
    got = decode_attention(q[-1:].cuda(), k, v, table.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"))
    want, bound = oracle.attend(q[-1:], kk, vv, dtype=torch.bfloat16)
    _close(got, want, bound)


# ---- prompts that are shared out over the chip --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [(torch.bfloat16, 2, 1, 64, 64), (torch.float16, 16, 2, 64, 256), (torch.float16, 1, 1, 128, 16),
                                                            (torch.float32, 4, 4, 64, 128), (torch.float32, 8, 1, 128, 0), (torch.bfloat16, 4, 2, 128, 0), (torch.bfloat16, 12, 2, 64, 256),
                                                            (torch.bfloat16, 16, 4, 128, 64), (torch.float16, 16, 4, 64, 16), (torch.bfloat16, 2, 1, 64, 24)])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 20000, 5), (False, 0, 0)])
def test_chunks_behind_long_caches(dtype, heads, kv_heads, dim, page, causal, window, sinks):
    """Few tiles of rows with many keys: their work is cut anywhere and joined.  Rows at the ends and borders of tiles are compared."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    if window and not causal:
        pytest.skip("a window needs causal order")
    print(dtype, heads, kv_heads, dim, page, causal, window, sinks, flush=True)
    g = _gen(21)
    new, totals = [130, 1, 300, 4, 257], [40000, 33001, 55013, 3, 257]
    dense, k, v, table = _paged(totals, kv_heads, dim, page or 64, dtype, g, spare=0)
    q = (1.5 * torch.randn(sum(new), heads, dim, generator=g)).to(dtype)
    dense[2][1][54900] = NAN  # seen by some rows only
    if page:
        bad = 54900 // page
        v[table[2, bad], 54900 % page] = NAN
        got = prompt_attention(q.cuda(), k, v, _starts(new).cuda(), block_tables=table.cuda(), context_lens=torch.tensor(totals, dtype=torch.int32, device="cuda"),
                               causal=causal, window=window, sinks=sinks)
    else:
        packed = [torch.cat([d[i] for d in dense]).cuda() for i in range(2)]
        got = prompt_attention(q.cuda(), *packed, _starts(new).cuda(), cu_seqlens_k=_starts(totals).cuda(), causal=causal, window=window, sinks=sinks)
    at = 0
    for s, n in enumerate(new):
        for i in sorted({0, 1, 127, 128, 129, 186, 187, 255, 256, n - 2, n - 1} & set(range(n))):
            place = totals[s] - n + i
            upto = place + 1 if causal else totals[s]
            if upto <= 0:
                assert not got[at + i].any()
                continue
            first = max(0, place + 1 - window) if window else 0
            keys = [*range(min(sinks, first)), *range(first, upto)]
            want, bound = oracle.attend(q[at + i : at + i + 1], dense[s][0][keys], dense[s][1][keys], False, dtype=dtype)
            _close(got[at + i : at + i + 1], want, bound, (s, i))
        at += n


# ---- prompts ---------------------------------------------------------------------------------------------------------


def _starts(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.bfloat16, 16, 2, 64), (torch.float16, 2, 1, 128), (torch.float32, 2, 2, 64)])
@pytest.mark.parametrize("totals", [[0, 30000, 0, 0, 28000, 0], [0, 0, 33000], [25000, 0]])
def test_rows_without_keys_among_long_caches(dtype, heads, kv_heads, dim, totals):
    """They have no part in the list of tiles of keys that is shared out, and are written all the same."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(dtype, heads, kv_heads, dim, totals, flush=True)
    g = _gen(26)
    new = [70 + 5 * s for s in range(len(totals))]
    dense, k, v, table = _paged(totals, kv_heads, dim, 64, dtype, g, spare=0)
    q = (1.5 * torch.randn(sum(new), heads, dim, generator=g)).to(dtype)
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    prompt_attention(q.cuda(), k, v, _starts(new).cuda(), block_tables=table.cuda(), context_lens=torch.tensor(totals, dtype=torch.int32, device="cuda"), out=out)
    at = 0
    for s, n in enumerate(new):
        if totals[s] == 0:
            assert not out[at : at + n].any(), s
        else:
            for i in (0, 31, 32, n - 1):
                upto = totals[s] - n + i + 1
                want, bound = oracle.attend(q[at + i : at + i + 1], dense[s][0][:upto], dense[s][1][:upto], False, dtype=dtype)
                _close(out[at + i : at + i + 1], want, bound, (s, i))
        at += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (2, 2, 128), (7, 1, 64), (2, 1, 96), (16, 4, 64), (12, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 33, 0), (True, 70, 4), (True, 1, 130), (False, 0, 0)])
def test_prompts_of_every_length(dtype, heads, kv_heads, dim, causal, window, sinks):
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(dtype, heads, kv_heads, dim, causal, window, sinks, flush=True)
    g = _gen(11)
    lens = [1, 0, 31, 32, 65, 129, 2, 260]
    starts = _starts(lens)
    total, behind = sum(lens), 5
    q = (1.5 * torch.randn(total + behind, heads, dim, generator=g)).to(dtype)
    k, v = (torch.randn(total, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    out = torch.full((total + behind, heads, dim), 7.0, dtype=dtype, device="cuda")
    prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts.cuda(), causal=causal, window=window, sinks=sinks, out=out)
    assert (out[total:] == 7.0).all()
    for s in range(len(lens)):
        at = slice(int(starts[s]), int(starts[s + 1]))
        want, bound = oracle.attend(q[at], k[at], v[at], causal, window, sinks, dtype=dtype)
        _close(out[at], want, bound, lens[s])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (3, 1, 128, 256), (2, 2, 64, 48), (2, 1, 64, 9), (16, 4, 64, 64), (8, 4, 128, 16),
                                                     (2, 1, 128, 24), (16, 2, 64, 8)])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 100, 3), (False, 0, 0)])
def test_chunks_behind_cached_rows(dtype, heads, kv_heads, dim, page, causal, window, sinks):
    """New rows behind what is cached, a row without any, more rows than keys (the first of them see nothing)."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(dtype, heads, kv_heads, dim, page, causal, window, sinks, flush=True)
    g = _gen(12)
    new, totals = [1, 70, 0, 130, 5, 40], [200, 333, 50, 130, 2, 0]
    starts = _starts(new)
    dense, k, v, table = _paged(totals, kv_heads, dim, page, dtype, g)
    q = (1.5 * torch.randn(sum(new), heads, dim, generator=g)).to(dtype)
    got = prompt_attention(q.cuda(), k, v, starts.cuda(), block_tables=table.cuda(), context_lens=torch.tensor(totals, dtype=torch.int32, device="cuda"),
                           causal=causal, window=window, sinks=sinks)
    packed_starts = _starts(totals)
    packed = [torch.cat([d[i] for d in dense]).cuda() for i in range(2)]
    other = prompt_attention(q.cuda(), *packed, starts.cuda(), cu_seqlens_k=packed_starts.cuda(), causal=causal, window=window, sinks=sinks)
    for s in range(len(new)):
        at = slice(int(starts[s]), int(starts[s + 1]))
        want, bound = oracle.attend(q[at], *dense[s], causal, window, sinks, dtype=dtype)
        _close(got[at], want, bound, ("pages", s))
        _close(other[at], want, bound, ("packed", s))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 64), (32, 1, 128), (8, 1, 64), (64, 2, 64), (24, 3, 128), (4, 1, 64), (6, 3, 64)])
@pytest.mark.parametrize("new,longest", [([1, 0, 3, 2, 40, 1, 5, 16, 17, 33, 4, 1], 300), ([2, 1, 1], 300), ([1, 3, 1, 9], 12000), ([5, 1, 7, 30], 9000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3)])
def test_few_rows_of_many_heads(dtype, heads, kv_heads, dim, new, longest, window, sinks):
    """A tile holds several heads of few rows, in wavefronts of two, four and eight heads; a value that some rows see is NaN."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(dtype, heads, kv_heads, dim, new, longest, window, sinks, flush=True)
    g = _gen(28)
    totals = [min(longest, n + longest * (s + 1) // len(new)) if s != 1 else new[1] for s, n in enumerate(new)]
    dense, k, v, table = _paged(totals, kv_heads, dim, 64, dtype, g)
    q = (1.5 * torch.randn(sum(new), heads, dim, generator=g)).to(dtype)
    last = len(new) - 1
    at = totals[last] - 1
    dense[last][1][at, 0, 5] = NAN
    v[table[last, at // 64], at % 64, 0, 5] = NAN
    got = prompt_attention(q.cuda(), k, v, _starts(new).cuda(), block_tables=table.cuda(), context_lens=torch.tensor(totals, dtype=torch.int32, device="cuda"),
                           window=window, sinks=sinks)
    packed = [torch.cat([d[i] for d in dense]).cuda() for i in range(2)]
    other = prompt_attention(q.cuda(), *packed, _starts(new).cuda(), cu_seqlens_k=_starts(totals).cuda(), window=window, sinks=sinks)
    row = 0
    for s, n in enumerate(new):
        for i in range(n):
            upto = totals[s] - n + i + 1
            first = max(0, upto - window) if window else 0
            keys = [*range(min(sinks, first)), *range(first, upto)]
            want, bound = oracle.attend(q[row : row + 1], dense[s][0][keys], dense[s][1][keys], False, dtype=dtype)
            _close(got[row : row + 1], want, bound, ("pages", s, i))
            _close(other[row : row + 1], want, bound, ("packed", s, i))
            row += 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 5, 8, 9, 16, 24, 48, 64, 256])
def test_prompts_leave_pages_outside_the_cache_unread(page, dim, dtype):
    """Their keys are hidden, in the middle, at the end and where all of them are; pages that end inside tiles of 64 keys."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(page, dim, dtype, flush=True)
    g = _gen(27)
    new, totals = [40, 70, 3, 33], [200, 333, 90, 600]
    dense, k, v, table = _paged(totals, 2, dim, page, dtype, g)
    q = (1.5 * torch.randn(sum(new), 4, dim, generator=g)).to(dtype)
    bad = {0: [0], 1: [(totals[1] - 1) // page], 2: list(range(-(-totals[2] // page))), 3: [i for i in range(-(-totals[3] // page)) if 100 <= i * page <= 140]}
    for s, pages in bad.items():
        for i, n in enumerate(pages):
            table[s, n] = -1 if i % 2 == 0 else k.size(0)
    got = prompt_attention(q.cuda(), k, v, _starts(new).cuda(), block_tables=table.cuda(), context_lens=torch.tensor(totals, dtype=torch.int32, device="cuda"))
    at = 0
    for s, n in enumerate(new):
        for i in range(n):
            keys = [j for j in range(totals[s] - n + i + 1) if j // page not in bad[s]]
            if not keys:
                assert not got[at + i].any()
                continue
            want, bound = oracle.attend(q[at + i : at + i + 1], dense[s][0][keys], dense[s][1][keys], False, dtype=dtype)
            _close(got[at + i : at + i + 1], want, bound, (s, i))
        at += n


@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (16, 4)])
@pytest.mark.parametrize("sequences", [63, 64, 65, 200])
def test_many_short_prompts(sequences, heads, kv_heads):
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(sequences, heads, kv_heads, flush=True)
    g = _gen(22)
    lens = torch.randint(0, 40, (sequences,), generator=g).tolist()
    lens[0], lens[-1], lens[sequences // 2] = 0, 33, 150
    starts = _starts(lens)
    q = (1.5 * torch.randn(sum(lens), heads, 64, generator=g)).to(torch.bfloat16)
    k, v = (torch.randn(sum(lens), kv_heads, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts.cuda())
    for s in range(sequences):
        at = slice(int(starts[s]), int(starts[s + 1]))
        want, bound = oracle.attend(q[at], k[at], v[at], True, dtype=torch.bfloat16)
        _close(got[at], want, bound, (s, lens[s]))


def test_starts_that_run_backwards_stay_inside_the_workspace():
    """Sequences that lie on one another, 3 x 94 tiles of 32 rows where the rows make room for 98.  The launch has places for 192 of them and takes the last
    of each sequence first: the rows of tiles 30 to 93, whose answer is one since all three sequences have the same keys."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    g, n, total, page = _gen(25), 3000, 6000, 64
    dense, k, v, table = _paged([total], 2, 64, page, torch.bfloat16, g)
    q = (1.5 * torch.randn(n, 16, 64, generator=g)).to(torch.bfloat16)
    starts = torch.tensor([0, n, 0, n, 0, n], dtype=torch.int32, device="cuda")
    lens = torch.full((5,), total, dtype=torch.int32, device="cuda")
    got = prompt_attention(q.cuda(), k, v, starts, block_tables=table.cuda().expand(5, -1).contiguous(), context_lens=lens)
    for i in (960, 991, 992, 1500, n - 1):
        upto = total - n + i + 1
        want, bound = oracle.attend(q[i : i + 1], dense[0][0][:upto], dense[0][1][:upto], False, dtype=torch.bfloat16)
        _close(got[i : i + 1], want, bound, i)


def test_tens_of_thousands_of_prompts_of_a_token_or_none():
    """A single token's output is its value."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    g = _gen(24)
    lens = torch.randint(0, 2, (70000,), generator=g)
    n = int(lens.sum())
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32).cuda()
    q, k, v = (torch.randn(n, h, 64, generator=g).to(torch.bfloat16).cuda() for h in (6, 3, 3))
    got = prompt_attention(q, k, v, starts)
    assert torch.equal(got, v.repeat_interleave(2, dim=1))


@pytest.mark.parametrize("sequences,behind", [(40, 0), (2, 0), (64, 20)])
def test_more_tiles_than_the_chip_holds_at_once(sequences, behind):
    """They start in the order of what they cost; `behind`: keys of every sequence in front of its rows."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    print(sequences, behind, flush=True)
    g = _gen(23)
    heads, kv_heads, dim = 16, 4, 128
    lens = torch.randint(0, 300 if sequences > 2 else 3000, (sequences,), generator=g).tolist()
    lens[-1] = 2500 if sequences == 2 else 1
    lens[sequences // 2] += 2048
    totals = [n + behind for n in lens]
    starts, key_starts = _starts(lens), _starts(totals)
    assert sum((n + 31) // 32 for n in lens) > 128
    q = (1.5 * torch.randn(sum(lens), heads, dim, generator=g)).to(torch.float16)
    k, v = (torch.randn(sum(totals), kv_heads, dim, generator=g).to(torch.float16) for _ in range(2))
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts.cuda(), cu_seqlens_k=key_starts.cuda()).cpu()
    assert torch.isfinite(got).all()
    for s, n in enumerate(lens):
        for i in sorted({0, 31, 32, 63, 64, 100, n // 2, n - 1} & set(range(n))):
            row, keys = slice(int(starts[s]) + i, int(starts[s]) + i + 1), slice(int(key_starts[s]), int(key_starts[s]) + behind + i + 1)
            want, bound = oracle.attend(q[row], k[keys], v[keys], False, dtype=torch.float16)
            _close(got[row], want, bound, (s, n, i))


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_a_row_does_not_see_does_not_reach_it(dtype, dim):
    """NaN and infinities in keys and values: the rows that see them are NaN, the others as if they were not there."""
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    g = _gen(13)
    n, heads = 150, 2
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dtype) for h in (heads, 1, 1))
    starts = _starts([n]).cuda()
    clean = prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts, window=40, sinks=2)
    for at, value in ((100, NAN), (100, float("inf")), (1, NAN), (20, float("-inf"))):
        for name in ("v", "k"):
            kk, vv = k.clone(), v.clone()
            (vv if name == "v" else kk)[at] = value
            got = prompt_attention(q.cuda(), kk.cuda(), vv.cuda(), starts, window=40, sinks=2)
            sees = torch.tensor([at in oracle.visible(i, n, True, 40, 2) for i in range(n)])
            for i in range(n):
                if not sees[i]:
                    want, bound = oracle.attend(q[i : i + 1], k[: i + 1], v[: i + 1], True, 40, 2, dtype=dtype)
                    _close(got[i : i + 1], want, bound, (name, at, value, i))
            assert not torch.isfinite(got.cpu()[sees]).all() and torch.equal(torch.isfinite(clean), torch.ones_like(clean, dtype=torch.bool))


def test_prompts_with_other_strides_and_off_alignment():
    from nanovllm_voxcpm_amd.attention_ops import prompt_attention

    g = _gen(14)
    n, heads, dim = 77, 2, 64
    for dtype in DTYPES:
        qkv = torch.randn(n, 3 * heads * dim, generator=g).to(dtype).cuda()
        q, k, v = (p.view(n, heads, dim) for p in qkv.chunk(3, dim=1))
        starts = _starts([n]).cuda()
        want, bound = oracle.attend(q.cpu(), k.cpu(), v.cpu(), dtype=dtype)
        _close(prompt_attention(q, k, v, starts), want, bound)
        odd = [torch.empty(n * heads * dim + 1, dtype=dtype, device="cuda")[1:].view(n, heads, dim).copy_(t) for t in (q, k, v)]
        _close(prompt_attention(*odd, starts), want, bound)
        turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        out = torch.empty(heads, n, dim, dtype=dtype, device="cuda").transpose(0, 1)
        prompt_attention(*turned, starts, out=out)
        _close(out, want, bound)


# ---- host paths, streams and graphs ----------------------------------------------------------------------------------------


def _everything(seed, dtype, out=None):
    """One call of every kind: the step of a batch of prompts and the step behind it."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotary_table, rotate_qk

    g = _gen(seed)
    t, heads, kv_heads, dim, page = 93, 8, 2, 64, 16
    q, k, v, weights, _ = _rotation(t, heads, kv_heads, dim, dtype, seed)
    caches = [torch.zeros(12, page, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    slots = torch.arange(t, dtype=torch.int32, device="cuda")
    tables = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)[:1].contiguous()
    results = list(rotate_qk(q, k, slots, rotary_table(dim, 128).cuda(), q_weight=weights[0], k_weight=weights[1]))
    turned, _ = rotate_qk(q, k, slots, rotary_table(dim, 128).cuda(), interleaved=True, v=v, k_cache=caches[0], v_cache=caches[1], slot_mapping=slots)
    starts = _starts([40, t - 40]).cuda()
    results += [turned, *caches, prompt_attention(turned, results[1], v, starts, window=30, sinks=2), prompt_attention(turned, results[1], v, starts, causal=False, scale=0.3),
                prompt_attention(turned, *caches, _starts([t]).cuda(), block_tables=tables, context_lens=torch.tensor([t], dtype=torch.int32, device="cuda")),
                decode_attention(turned[-1:], *caches, tables, torch.tensor([t], dtype=torch.int32, device="cuda"), sinks=3, window=50)]
    return results


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_host_paths_make_the_same_calls(dtype, monkeypatch):
    from nanovllm_voxcpm_amd import _hip

    if _hip.load_fastcall() is None:
        pytest.skip("the C++ host path is not built (make -C nanovllm-voxcpm_amd/csrc fastcall)")
    quick = _everything(30, dtype)
    monkeypatch.setenv("MLORA_NO_FASTCALL", "1")
    _hip.reload_knobs()
    assert _hip.load_fastcall() is None
    slow = _everything(30, dtype)
    assert len(quick) == len(slow) and all(torch.equal(a, b) for a, b in zip(quick, slow))


def test_the_quick_host_path_leaves_what_it_does_not_know_to_the_other():
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotate_qk

    q, k = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")
    table = torch.zeros(4, 64, device="cuda")
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="differ"):
        rotate_qk(q, k[:2], positions, table)
    with pytest.raises(ValueError, match="positions lives on cpu"):
        rotate_qk(q, k, positions.cpu(), table)
    with pytest.raises(RuntimeError, match="no backward"):
        rotate_qk(q.clone().requires_grad_(), k, positions, table)
    with torch.no_grad():
        rotate_qk(q.clone().requires_grad_(), k, positions, table)
    with pytest.raises(RuntimeError, match="rotary = 24"):
        rotate_qk(q, k, positions, table[:, :24])
    with pytest.raises(ValueError, match="evenly"):
        prompt_attention(q, k[:, :1].expand(3, 3, 64).contiguous(), k[:, :1].expand(3, 3, 64).contiguous(), positions)
    cache = torch.zeros(2, 16, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="negative"):
        decode_attention(q, cache, cache, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), positions, window=-1)
    with pytest.raises(ValueError, match="context_lens"):
        decode_attention(q, cache, cache, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), positions.long())
    assert decode_attention(q[:0], cache, cache, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), positions[:0]).shape == (0, 4, 64)
    assert prompt_attention(q[:0], k[:0], k[:0], positions[:1]).shape == (0, 4, 64)
    assert not decode_attention(q + 1, cache, cache, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), positions + 5).any()  # a table without pages


def test_calls_on_another_stream_and_two_at_once():
    streams = [torch.cuda.Stream() for _ in range(3)]
    want = [[t.clone() for t in _everything(40 + i, torch.bfloat16)] for i in range(3)]
    torch.cuda.synchronize()
    got = []
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            got.append(_everything(40 + i, torch.bfloat16))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("longest,dim", [(700, 64), (30000, 64), (9000, 128)])
def test_graphs_of_decode_and_chunks_replayed(longest, dim):
    """Two graphs, replayed in turn with eager work between the replays; lengths, pages and values change in place."""
    from nanovllm_voxcpm_amd.attention_ops import decode_attention, prompt_attention, rotary_table, rotate_qk

    g = _gen(50)
    page, heads, kv_heads, sequences, chunk = 64, 8, 2, 3, 70
    pages = -(-longest // page)
    caches = [torch.randn(sequences * pages, page, kv_heads, dim, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    tables = torch.arange(sequences * pages, dtype=torch.int32, device="cuda").view(sequences, pages).contiguous()
    lens = torch.tensor([longest, 5, longest // 2], dtype=torch.int32, device="cuda")
    rows = torch.randn(sequences + chunk, heads + 2 * kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
    starts, chunk_lens = _starts([chunk]).cuda(), torch.tensor([longest], dtype=torch.int32, device="cuda")
    slots = torch.full((sequences + chunk,), -1, dtype=torch.int32, device="cuda")
    slots[:3] = torch.tensor([longest - 1, pages * page + 4, 2 * pages * page + longest // 2 - 1], dtype=torch.int32)
    table = rotary_table(dim, 64).cuda()
    positions = torch.zeros(sequences + chunk, dtype=torch.int32, device="cuda")

    def step():
        q, k, v = rows.split([heads, kv_heads, kv_heads], dim=1)
        q, _ = rotate_qk(q, k, positions, table, v=v, k_cache=caches[0], v_cache=caches[1], slot_mapping=slots)
        return [decode_attention(q[:sequences], *caches, tables, lens, window=0), decode_attention(q[:sequences], *caches, tables, lens, window=333, sinks=4),
                prompt_attention(q[sequences:], *caches, starts, block_tables=tables, context_lens=chunk_lens)]

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for i in range(5):
        rows.copy_(torch.randn(rows.shape, generator=g).to(torch.bfloat16))
        positions.fill_(7 * i % 64)
        lens.copy_(torch.tensor([longest - i, 5 + i, longest // 2 + 3 * i], dtype=torch.int32))
        graph, held = graphs[i % 2]
        graph.replay()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
