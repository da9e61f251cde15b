"""The serving operators at their edges: scales, codes, queries and devices that
ordinary use seldom meets, against the plain 64-bit forms."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from xpose_b200 import serving as S  # noqa: E402

F16, I8 = torch.float16, torch.int8


def test_tensors_of_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    outs = []
    for device in ("cuda:0", "cuda:1"):
        torch.cuda.set_device(0)
        g = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(70, h, 64, generator=g).to(F16).to(device) for h in (4, 1, 1))
        pos = torch.arange(70, dtype=torch.int32, device=device)
        slots = torch.arange(70, device=device)
        turns, _ = S.rope_turns(64, 1e4, device=device)
        pages = S.new_pages(8, 16, 1, 64, I8, device=device)
        scratch = S.new_scratch(device)
        one = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        S.rope_rows(q, q, pos, turns)
        S.kv_write(*pages, k, v, slots, positions=pos, turns=turns)
        a, b = torch.empty_like(q), torch.empty_like(q)
        S.attention_packed(a, q, k, v, one(0, 70), scratch)
        S.attention_paged(b, q, *pages, one(0, 1, 2, 3, 4)[None].contiguous(), one(70), one(0, 70), 70, scratch)
        assert S.error_word(scratch) == 0 and torch.cuda.current_device() == 0
        outs.append((a.cpu(), b.cpu()))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
