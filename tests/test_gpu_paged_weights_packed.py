"""Attention weights of packed steps, some of whose sequences generate while others take chunks, over e4m3 keys whose scales are no powers of
two: each sequence's scores are those that its lse was made of.  Against the 64-bit restatement (oracle/paged_oracle.py)."""
import pytest
import torch

import mercury_artifact_amd as M
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Setting:
    """A cache of random codes with any positive scales, and no key that has none."""

    def __init__(self, lengths, Hkv, D, page, seed):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lengths, self.page = lengths, page
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts)
        order, at = torch.randperm(pages, generator=g).tolist(), 0
        self.table = []
        for c in counts:
            self.table.append(order[at:at + c] + [-1] * (max(counts) - c))
            at += c
        codes = torch.randn(2, pages, page, Hkv, D, generator=g).to(E4M3)
        self.scale = torch.rand(2, pages, page, Hkv, generator=g) * 0.9 + 0.55
        self.values = codes.double() * self.scale.double()[..., None]
        self.cache, self.scales = codes.cuda(), self.scale.cuda()
        self.weights = M.paged_weights(pages, page, Hkv)

    def tables(self):
        return _ints(self.table), _ints(self.lengths)


@pytest.mark.parametrize("lengths,new,Hq,Hkv,D", [
    ([400, 260, 700, 90, 33], [1, 70, 2, 0, 1], 8, 2, 64),
    ([300, 129, 257], [1, 33, 1], 16, 1, 128),                   # 16 rows, 528, 16
    ([150, 200, 31], [1, 20, 2], 20, 1, 96),                     # 20 rows, 400, 40: the second kernel's alone from 33 on
    ([90, 140], [1, 3], 40, 1, 64),                              # 40 rows, 120
    ([500], [1], 4, 1, 64),
])
def test_scores_are_those_of_the_sequences_lse(lengths, new, Hq, Hkv, D):
    s = Setting(lengths, Hkv, D, 16, seed=Hq)
    G = Hq // Hkv
    few = 16 if G <= 16 else 32 if G <= 32 else 64       # rows of a sequence and K/V head whose scores take the scales in fp32
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    q = torch.randn(starts[-1], Hq, D, generator=s.g).bfloat16()
    exact = torch.cat([l for _, l, _, _ in P.paged_attention(q, s.values, s.table, lengths, D ** -0.5, True, None, starts)], 1).float()
    for most in (None, max(new)):
        got = M.paged_attn_weights(q.cuda(), s.cache, *s.tables(), D ** -0.5, exact.cuda(), s.weights, scales=s.scales, starts=_ints(starts),
                                   most_new=most, decay=0.0, out=torch.zeros_like(s.weights)).cpu()
        want, off = P.paged_weights(q, s.values, s.table, lengths, D ** -0.5, exact, s.weights.cpu(), True, starts, 0.0)
        _, lse = M.paged_attn_fwd(q.cuda(), s.cache, *s.tables(), D ** -0.5, scales=s.scales, starts=_ints(starts), most_new=most)
        own = M.paged_attn_weights(q.cuda(), s.cache, *s.tables(), D ** -0.5, lse, s.weights, scales=s.scales, starts=_ints(starts),
                                   most_new=most, decay=0.0, out=torch.zeros_like(s.weights)).cpu().double()
        for b, n in enumerate(lengths):
            page, slot = torch.tensor(s.table[b])[torch.arange(n) // 16], torch.arange(n) % 16
            if new[b] * G <= few:
                assert ((got[page, slot].double() - want[page, slot]).abs() <= off[page, slot]).all(), b
            # Every row's weights add up to one: its scores and those behind its lse are sums of the same products in fp32, each off by less than
            # |q| |k| scale (D + 4) 2^-24 < 2^-12 here, and so is the sum of n weights, by 2^-12 too.
            for h in range(Hkv):
                assert abs(own[page, slot, h].sum().item() - new[b] * G) <= new[b] * G * 2.0 ** -10, (b, h)
