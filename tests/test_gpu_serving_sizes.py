"""Sizes past 31 bits are refused by the serving operators' wrappers: the C-ABI takes them as 32-bit ints, which would drop the
bits above. (Views of one element repeated: nothing of that size is allocated.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    torch.cuda.set_device(0)


def test_sizes_past_31_bits_are_refused():
    from wfamd import ops
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for page in (2 ** 32 + 32, 2 ** 31, -2 ** 32 + 32):
        with pytest.raises(ValueError, match="kv_page_plan"):
            ops.kv_page_plan(i, i, i, table, 2, page_size=page)
    with pytest.raises(ValueError, match="kv_page_plan"):
        ops.kv_page_plan(i, i, i, table, 2 ** 32 + 2)
    freqs, _ = ops.rotary_frequencies(64)
    q = torch.zeros(2, 1, 64, device="cuda")
    with pytest.raises(ValueError, match="rotary_embed"):
        ops.rotary_embed(q.expand(2, 2 ** 32 + 1, 64), None, i, freqs)
    with pytest.raises(ValueError, match="rotary_embed"):
        ops.rotary_embed(q, q.expand(2, 2 ** 32 + 1, 64), i, freqs)
    with pytest.raises(ValueError, match="token_logprobs"):
        ops.token_logprobs(torch.zeros(1, 1, device="cuda").expand(1, 2 ** 32 + 7))
    with pytest.raises(ValueError, match="token_logprobs"):
        ops.token_logprobs(torch.zeros(1, 2, device="cuda", dtype=torch.bfloat16).expand(2 ** 32 + 1, 2))
    pool = torch.zeros(1, 1, 4096, dtype=torch.bfloat16, device="cuda")
    a = dict(q=torch.zeros(2, 1, 128, device="cuda"), k_pool=pool, v_pool=pool, page_table=table, seq_lens=i, prefix_rows=i, prefix_lens=i)
    ops.shared_prefix_attention(**a)
    for kw in (dict(k_pool=pool.expand(2 ** 32 + 1, 1, 4096), v_pool=pool.expand(2 ** 32 + 1, 1, 4096)),
               dict(q=a["q"].expand(2, 2 ** 32 + 1, 128))):
        with pytest.raises(ValueError, match="shared_prefix_attention"):
            ops.shared_prefix_attention(**{**a, **kw})
