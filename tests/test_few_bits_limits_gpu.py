"""Few-bit serving operators (K16, K17) at the limits of what their documentation allows, each against its definition in 64 bits."""
import math

import pytest
import torch

from adt_str_amd import kernels as K
from tests.test_few_bits_gpu import check_attn, check_held, gen, kv_rows

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_len,cap,lens", [
    (2, 2, 4, 100, [103, 100, 101, 99, 2 ** 31 - 1, -3]),                     # the newest rows lie behind the cache; a length no cache has
    (6, 2, 9, 33, [40, 41, 42, 33, 5]), (1, 1, 40, 64, [70, 64, 103, 104]),   # several blocks of rows, some of which see all, some less
    (4, 1, 3, 3000, [3001, 3002, 2999])])                                     # cut into spans
@pytest.mark.parametrize("causal", [True, False])
def test_attn_kv4_lengths_past_the_capacity(dim, heads, kv_heads, q_len, cap, lens, causal):
    """``key_len`` is the sequence's length, whatever part of it the cache holds: causal query i sees the first min(capacity, key_len - (q_len - 1 - i))
    positions."""
    batch = len(lens)
    k, v = kv_rows(batch * cap, kv_heads, dim, cap + q_len)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    K.kv4_append(c, k, v)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (1.5 * torch.randn(batch * q_len, heads * dim, generator=gen(7))).to(BF16).cuda()
    scale = 1.0 / math.sqrt(dim)
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=scale, q_len=q_len, causal=causal, want_lse=True)
    check_attn(out, lse, q, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, q_len, lens, scale, causal)


def test_append_and_causal_attention_of_a_sequence_that_outgrows_its_cache():
    """The chunk's rows that do not fit are left out by the append and seen by nobody; its queries see what their positions say."""
    heads, dim, cap, q_len, end = 2, 128, 50, 6, 53
    k, v = kv_rows(end, heads, dim, 4)
    c = K.KV4Cache(1, cap, heads, dim)
    at = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    K.kv4_append(c, k[:end - q_len], v[:end - q_len], at(end - q_len))
    K.kv4_append(c, k[end - q_len:], v[end - q_len:], at(end))
    held = K.kv4_read(c, out_dtype=torch.float32)
    check_held(held[0], k[:cap], heads, dim)
    check_held(held[1], v[:cap], heads, dim)
    q = torch.randn(q_len, heads * dim, generator=gen(9)).to(BF16).cuda()
    out, lse = K.attn_kv4(q, c, at(end), heads=heads, scale=dim ** -0.5, q_len=q_len, causal=True, want_lse=True)
    check_attn(out, lse, q, k[None, :cap], v[None, :cap], heads, heads, dim, 1, q_len, [end], dim ** -0.5, True)
