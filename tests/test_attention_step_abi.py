"""Refusals of the attention step's entry points (no GPU needed): every check is made on the host before a CUDA call."""
import pytest

import pfng_b200 as pb

OK, INVALID, SHAPE, ALIGN = 0, -1, -2, -3
FAKE = 0x10000  # never dereferenced: every call below is rejected, or empty, on the host


@pytest.fixture(scope="module")
def L():
    return pb.lib()


def changed(base, **kw):
    args = dict(base)
    args.update(kw)
    return list(args.values())


def test_cache_bytes():
    assert pb.kv_cache_bytes(3, 16, 2, 128) == 3 * 2 * 16 * (64 + 8)
    assert pb.kv_cache_bytes(1, 64, 8, 64) == 8 * 64 * 36
    assert pb.kv_cache_bytes(1 << 20, 64, 8, 128) == (1 << 29) * 72  # past 32 bits
    for bad in ((0, 16, 1, 128), (1, 8, 1, 128), (1, 24, 1, 128), (1, 16, 0, 128), (1, 16, 1, 48)):
        assert pb.kv_cache_bytes(*bad) == 0


PLAN = dict(kv_len=FAKE, q_len=FAKE, requests=2, block_table=FAKE, max_pages=4, free_pages=FAKE, num_free=3,
            page_size=16, seq_len=FAKE, cu_q=FAKE, positions=FAKE, slots=FAKE, max_tokens=5, counts=FAKE, stream=None)


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(requests=-1)), (INVALID, dict(max_pages=-1)), (INVALID, dict(num_free=-1)),
    (INVALID, dict(max_tokens=-1)), (SHAPE, dict(page_size=0)), (SHAPE, dict(page_size=24)),
    (SHAPE, dict(max_tokens=1 << 31)), (INVALID, dict(kv_len=None)), (INVALID, dict(q_len=None)),
    (INVALID, dict(block_table=None)), (INVALID, dict(free_pages=None)), (INVALID, dict(seq_len=None)),
    (INVALID, dict(cu_q=None)), (INVALID, dict(positions=None)), (INVALID, dict(slots=None)),
    (INVALID, dict(counts=None)), (ALIGN, dict(kv_len=FAKE + 2)), (ALIGN, dict(slots=FAKE + 4)),
    (ALIGN, dict(block_table=FAKE + 1))])
def test_plan_refusals(L, status, change):
    assert L.pfng_b200_kv_plan(*changed(PLAN, **change)) == status


ROPE = dict(x=FAKE, in_format=0, ldx=384, q_weight=None, k_weight=None, eps=1e-6, positions=FAKE, cos_sin=FAKE,
            max_pos=100, rot_dim=64, interleaved=0, q_out=FAKE, ldq=256, k_out=FAKE, ldk=128, out_format=2, tokens=3,
            heads_q=4, heads_k=2, head_dim=64, stream=None)


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(in_format=3)), (INVALID, dict(out_format=-1)), (INVALID, dict(tokens=-1)),
    (INVALID, dict(heads_k=-1)), (SHAPE, dict(head_dim=63)), (SHAPE, dict(head_dim=0)), (SHAPE, dict(head_dim=514)),
    (SHAPE, dict(rot_dim=66)), (SHAPE, dict(rot_dim=7)), (INVALID, dict(rot_dim=-2)), (SHAPE, dict(ldx=383)),
    (SHAPE, dict(ldq=255)), (SHAPE, dict(ldk=127)), (INVALID, dict(x=None)), (INVALID, dict(positions=None)),
    (INVALID, dict(cos_sin=None)), (INVALID, dict(q_out=None)), (INVALID, dict(k_out=None)), (ALIGN, dict(x=FAKE + 2)),
    (ALIGN, dict(q_out=FAKE + 1)), (ALIGN, dict(q_weight=FAKE + 2)), (OK, dict(tokens=0, x=None)),
    (OK, dict(heads_q=0, heads_k=0, x=None))])
def test_rope_refusals(L, status, change):
    assert L.pfng_b200_qk_norm_rope(*changed(ROPE, **change)) == status


APPEND = dict(k=FAKE, ldk=256, k_format=2, v=FAKE, ldv=256, v_format=0, slots=FAKE, k_cache=FAKE, v_cache=FAKE,
              num_pages=4, page_size=16, tokens=3, heads_kv=2, head_dim=128, stream=None)


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(k_format=3)), (INVALID, dict(v_format=-1)), (INVALID, dict(tokens=-1)),
    (INVALID, dict(num_pages=-1)), (SHAPE, dict(head_dim=48)), (SHAPE, dict(head_dim=544)), (SHAPE, dict(page_size=20)),
    (SHAPE, dict(ldk=255)), (SHAPE, dict(ldv=255)), (INVALID, dict(k=None)), (INVALID, dict(v=None)),
    (INVALID, dict(slots=None)), (INVALID, dict(k_cache=None)), (ALIGN, dict(k=FAKE + 1)), (ALIGN, dict(v=FAKE + 2)),
    (ALIGN, dict(slots=FAKE + 4)), (ALIGN, dict(k_cache=FAKE + 8)), (ALIGN, dict(v_cache=FAKE + 8)),
    (OK, dict(tokens=0, k=None)), (OK, dict(num_pages=0, k=None))])
def test_append_refusals(L, status, change):
    assert L.pfng_b200_kv_append_q4_0(*changed(APPEND, **change)) == status


ATTN = dict(q=FAKE, ldq=512, q_format=2, k_cache=FAKE, v_cache=FAKE, num_pages=8, page_size=16, block_table=FAKE,
            max_pages=4, seq_len=FAKE, cu_q=FAKE, requests=2, tokens=3, max_q=2, max_kv=60, heads_q=4, heads_kv=2,
            head_dim=128, scale=0.1, causal=1, window=0, out=FAKE, ldo=512, out_format=2, lse=None, workspace=None,
            workspace_bytes=0, path=0, stream=None)


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(q_format=3)), (INVALID, dict(out_format=4)), (INVALID, dict(requests=-1)),
    (INVALID, dict(tokens=-1)), (INVALID, dict(max_q=-1)), (INVALID, dict(max_kv=-1)), (INVALID, dict(window=-1)),
    (INVALID, dict(window=5, causal=0)), (INVALID, dict(path=4)), (INVALID, dict(path=-1)), (SHAPE, dict(head_dim=48)),
    (SHAPE, dict(head_dim=288)), (SHAPE, dict(head_dim=0)), (SHAPE, dict(heads_q=5)), (SHAPE, dict(heads_kv=0)),
    (SHAPE, dict(page_size=8)), (SHAPE, dict(max_pages=1 << 28)), (SHAPE, dict(ldq=511)), (SHAPE, dict(ldo=511)),
    (INVALID, dict(q=None)), (INVALID, dict(out=None)), (INVALID, dict(k_cache=None)), (INVALID, dict(v_cache=None)),
    (INVALID, dict(block_table=None)), (INVALID, dict(seq_len=None)), (INVALID, dict(cu_q=None)),
    (ALIGN, dict(q=FAKE + 1)), (ALIGN, dict(k_cache=FAKE + 8)), (ALIGN, dict(lse=FAKE + 2)),
    (OK, dict(tokens=0, q=None)), (OK, dict(requests=0, q=None)), (OK, dict(max_q=0, q=None))])
def test_attention_refusals(L, status, change):
    assert L.pfng_b200_attention_q4_0(*changed(ATTN, **change)) == status


def test_binding_refuses_other_types():
    torch = pytest.importorskip("torch")
    with pytest.raises(pb.PfngError):
        pb._value_format(torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(pb.PfngError):
        pb._value_format(torch.zeros(4, 4).t())
    with pytest.raises(pb.PfngError):
        pb._value_tensor("q8_0", 1, 32, "cpu")
