"""evict_positions with new_acc in the same memory as acc: refused where they meet, right beside it."""
import pytest
import torch

import q8_reference as ref
from flashinfer_mlsys2026_dsa_b200 import evict_positions

pytestmark = pytest.mark.gpu


def totals(rows, cols):
    return torch.rand(rows, cols, generator=torch.Generator().manual_seed(cols)).cuda()


def test_new_totals_that_meet_the_old_ones_are_refused():
    both = totals(4, 300)
    lens = torch.full((4,), 200, dtype=torch.int32, device="cuda")
    before = both.clone()
    for acc, new in ((both, both[:, 1:]), (both[:, :200], both[:, 199:]), (both[:, 100:], both[:, :101]),
                     (both[:1].expand(4, 300), both[:, 200:])):
        with pytest.raises(ValueError, match="overlap"):
            evict_positions(acc, lens, 64, new_acc=new)
    flat = totals(1, 1000)[0]
    with pytest.raises(ValueError, match="overlap"):
        evict_positions(flat[:400].view(4, 100), lens, 64, new_acc=flat[340:340 + 4 * 64].view(4, 64))
    assert torch.equal(both, before)


def test_new_totals_beside_the_old_ones():
    """Columns of one buffer, in either order, and rows behind each other."""
    lens = torch.tensor([200, 30, 0, 199], dtype=torch.int32, device="cuda")
    for at, to in ((slice(0, 200), slice(200, 270)), (slice(70, 270), slice(0, 70))):
        both = totals(4, 270)
        acc = both[:, at].clone()
        keep, n = evict_positions(both[:, at], lens, 64, new_acc=both[:, to])
        want, want_n, want_t = ref.evict(acc.cpu(), lens.cpu(), 64, 0, 0)
        assert keep.tolist() == want and n.tolist() == want_n
        for r in range(4):
            assert both[r, to][:want_n[r]].tolist() == want_t[r] and (both[r, to][want_n[r]:] == 0).all()
        assert torch.equal(both[:, at], acc)
    flat = totals(1, 4 * 264)[0]
    acc = flat[:800].view(4, 200)
    keep, _ = evict_positions(acc, lens, 64, new_acc=flat[800:].view(4, 64))
    assert keep.tolist() == ref.evict(acc.cpu(), lens.cpu(), 64, 0, 0)[0]
