"""The paged operators' CPU forms at the ends of their integer arguments."""

import pytest
import torch

from _paged_ref import attend_ref, make_cache
from nanokv_amd.paged import PagedKV, append_paged, attend_paged, move_paged, read_paged

FAR = [2 ** 32 + 5, -2 ** 63, 2 ** 63 - 1, 2 ** 32, 2 ** 31, -2 ** 32 + 7]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)


def test_slots_past_32_bits_lie_outside_the_cache():
    for kv in ("bf16", "int8"):
        cache = make_cache(3, 2, 16, 64, kv, "cpu")
        was = PagedKV(*(None if t is None else t.clone() for t in cache))
        rows = torch.ones(len(FAR), 2, 64)
        append_paged(cache, rows, rows, torch.tensor(FAR))
        move_paged(cache, torch.tensor(FAR), torch.arange(len(FAR)))
        move_paged(cache, torch.arange(len(FAR)), torch.tensor(FAR))
        assert _same(cache, was)
        assert all(bool((t == 0).all()) for t in read_paged(cache, torch.tensor(FAR)))


def test_lengths_tables_and_starts_past_32_bits():
    cache = make_cache(5, 1, 16, 64, "bf16", "cpu")
    q = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    tables = torch.tensor([[3, 1], [0, 2]])
    full = attend_paged(q[:2], cache, tables, torch.tensor([32, 0]))
    assert torch.equal(attend_paged(q[:2], cache, tables, torch.tensor([2 ** 32 + 3, -2 ** 63 + 4])), full)
    far = torch.tensor([[3, 2 ** 32 + 1], [-2 ** 63, 2]])
    ref, mag = attend_ref(q[:2], cache, far, torch.tensor([32, 32]))
    got = attend_paged(q[:2], cache, far, torch.tensor([32, 32]))
    assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag).all())
    # starts past the rows are their end
    want = attend_paged(q, cache, tables, torch.tensor([20, 9]), starts=torch.tensor([1, 3, 4]))
    got = attend_paged(q, cache, tables, torch.tensor([20, 9]), starts=torch.tensor([1, 3, 2 ** 32 + 3]))
    assert torch.equal(got, want)


def test_trees_of_many_sequences_need_no_bound():
    """More than 64 rows in all, at most 64 new tokens each: max_new may be left out."""
    g = torch.Generator().manual_seed(3)
    cache = make_cache(9, 1, 16, 64, "bf16", "cpu")
    tables = torch.tensor([[3, 0, 5, 1, 8], [7, 6, 2, 4, 8]])
    lengths, starts = torch.tensor([75, 70]), torch.tensor([0, 64, 104])
    q = torch.randn(104, 2, 64, generator=g).bfloat16()
    masks = torch.randint(-2 ** 62, 2 ** 62, (104,), generator=g)
    got = attend_paged(q, cache, tables, lengths, starts=starts, tree=masks)
    assert torch.equal(got, attend_paged(q, cache, tables, lengths, starts=starts, max_new=64, tree=masks))
    assert not bool((got == 0).all(-1).any())
    with pytest.raises(ValueError, match="at most 64 tokens"):
        attend_paged(q, cache, tables, lengths, starts=starts, max_new=65, tree=masks)


def test_masks_of_32_bits_name_no_further_tokens():
    """int32 masks: bit 31 is token 31's, not that of all tokens behind it."""
    g = torch.Generator().manual_seed(4)
    cache = make_cache(4, 1, 16, 64, "bf16", "cpu")
    q = torch.randn(40, 2, 64, generator=g).bfloat16()
    masks = torch.randint(-2 ** 31, 2 ** 31, (40,), generator=g).int()
    tables, lengths = torch.tensor([[3, 1, 2, 0]]), torch.tensor([50])
    assert torch.equal(attend_paged(q, cache, tables, lengths, tree=masks),
                       attend_paged(q, cache, tables, lengths, tree=masks.long() & 0xffffffff))


def test_a_decoder_step_takes_64_bit_numbers():
    """Slots, tables, lengths and starts of 64 bits, padding's far outside: the step's rows are those of 32 bits."""
    from nanokv_amd.qwen3 import Qwen3Config, Qwen3ForCausalLM, init_random_
    model = Qwen3ForCausalLM(Qwen3Config(vocab_size=64, hidden_size=128, intermediate_size=192, num_hidden_layers=2,
                                         num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                         max_position_embeddings=512))
    init_random_(model, 3, std=0.2)
    ids, pos = torch.arange(6), torch.tensor([0, 1, 2, 0, 1, 0])
    slots, tables = torch.tensor([32, 33, 34, 0, 1, -1]), torch.tensor([[2, -1], [0, 1]])
    lengths, starts = torch.tensor([3, 2]), torch.tensor([0, 3, 5])
    out = []
    for far in (False, True):
        model.attach_paged(3, 16)
        s, t = slots.clone(), tables.clone()
        if far:
            s[5], t[0, 1] = 2 ** 32 + 40, 2 ** 32
        args = (s, t, lengths, starts) if far else (x.int() for x in (s, t, lengths, starts))
        s, t, n, at = args
        out.append(model.paged_step(ids, pos, s, t, n, starts=at, max_new=3))
        out.append(model.model.layers[1].self_attn.attn.paged_cache.k.clone())
    assert torch.equal(out[0][:5], out[2][:5]) and torch.equal(out[1], out[3])
