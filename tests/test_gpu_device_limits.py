"""Counts that do not fit the 32-bit numbers of the C calls are refused, not cut off: tensors whose rows lie on top of one another (stride 0) have as many as one likes, without the memory."""
import pytest
import torch

from nano_b200 import ops
from nano_b200.engine import NB200Error

pytestmark = pytest.mark.gpu
MANY = 2 ** 32 + 1


def test_counts_beyond_32_bits():
    one = torch.zeros(1, 1, device="cuda")
    number, number64 = (torch.zeros(1, dtype=t, device="cuda") for t in (torch.int32, torch.int64))
    pool = ops.kv4_cache(2, 1, 32)
    row = torch.zeros(1, 1, 32, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for f in (lambda: ops.token_logprobs(one.expand(MANY, 1), number64.expand(MANY)), lambda: ops.token_logprobs(one.expand(1, MANY), number), lambda: ops.token_logprobs(one.expand(1, 2 ** 31), number, top=3),
              lambda: ops.kv4_write(pool, row.expand(MANY, 1, 32), row.expand(MANY, 1, 32), number.expand(MANY)), lambda: ops.kv4_read(pool, number.expand(MANY)),
              lambda: ops.pages_copy([one.expand(MANY, 1)], [0], [1]), lambda: ops.kv4_read(pool[:1].expand(MANY, 1, 1280), number),
              lambda: ops.kv4_write(pool[:1].expand(1, MANY, 1280), row.expand(1, MANY, 32), row.expand(1, MANY, 32), number),
              lambda: ops.kv4_attention(row.expand(1, MANY, 1, 32), pool, number.view(1, 1), number), lambda: ops.kv4_attention(row.view(1, 1, 1, 32).expand(MANY, 1, 1, 32), pool, number.view(1, 1).expand(MANY, 1), number.expand(MANY))):
        with pytest.raises(NB200Error, match="too many|too large|contiguous"):
            f()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1 << 20, "a refused call made copies"
