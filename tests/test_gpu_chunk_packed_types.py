"""TQPagedAttention.forward_chunk in both types: float16 queries go to the kernel for few rows whatever their number, bfloat16 ones to
that for many rows or to both at once, so lengths, heads, batches and offsets are checked with either.  Tolerances as in
test_gpu_chunk.py; the last test says how near float16 results are in the mean."""
import math

import pytest
import torch

from tests.test_gpu_chunk import BF, FEW, FP, MANY, Batch, Packed, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 3, 2])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [FEW, MANY, MANY[:3] + FEW[-6:]], ids=["few", "many", "both"])
def test_lengths(dev, d, bits, dtype, lens):
    p = Packed(Batch(lens, 16, dev, 20 + bits), d, bits, 8, 2, dtype, dev, 400, primary=bits != 2)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("d,bits,heads,kv", [(64, 4, 3, 3), (64, 3, 14, 2), (64, 2, 33, 1), (64, 4, 130, 1), (128, 4, 5, 1), (128, 3, 66, 2), (128, 2, 300, 1),
                                             (256, 4, 7, 1), (256, 3, 130, 1), (256, 2, 3, 3)])
@pytest.mark.parametrize("block,index", [(16, torch.int64), (7, torch.int32)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [[(2, 90), (40, 150)], [(70, 150)]], ids=["mixed", "one"])
def test_heads_and_blocks(dev, d, bits, heads, kv, block, index, dtype, lens):
    """Groups that do not divide a tile, and groups of more heads than a tile has rows (128 at heads of 64 and 256, 256 at 128)."""
    p = Packed(Batch(lens, block, dev, heads, index), d, bits, heads, kv, dtype, dev, 410)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("seqs", [255, 257, 600])
@pytest.mark.parametrize("d,bits", [(64, 3), (128, 4)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_many_sequences(dev, seqs, d, bits, dtype):
    lens = [((0, 1, 3, 1)[i % 4] if i % 97 else 40, 20 + i % 90 + 40 * (i % 97 == 0)) for i in range(seqs)]
    p = Packed(Batch(lens, 16, dev, 21), d, bits, 4, 2, dtype, dev, 420)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("lens", [[(2, 60)], [(80, 90)], [(80, 90), (2, 60)]], ids=["few", "many", "both"])
@pytest.mark.parametrize("where", ["block", "place"])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_offsets_past_32_bits(dev, lens, where, dtype):
    """Rows and norms whose places do not fit 32 bits."""
    b = Batch(lens, 32, dev, 22, spare=0)
    p = Packed(b, 128, 4, 8, 2, dtype, dev, 430)
    steps = b.blocks - 1 if where == "block" else b.blocks * 32 - 1
    for name, last in (("k", 64), ("v", 64), ("kn", 1), ("vn", 1)):
        x = getattr(p, name)
        big = (1 << 32) // x.element_size() // steps // 64 * 64 + 128
        strides = ((big, 2 * last, last) if where == "block" else (32 * big, big, last)) + ((1,) if last > 1 else ())
        raw = torch.zeros(sum((s - 1) * t for s, t in zip(x.shape, strides)) + 1, dtype=x.dtype, device=dev)
        assert steps * big * x.element_size() > 1 << 32
        y = raw.as_strided(x.shape, strides)
        y.copy_(x)
        setattr(p, name, y)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("few,many", [(1, 40), (40, 1), (12, 12)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 3, 2])
def test_shares_of_a_mixed_batch(dev, few, many, d, bits):
    """bfloat16: workgroups divided between few and many rows (heads of 128 and 256), or one kernel after the other (64)."""
    b = Batch([(1 + i % 3, 100 + 177 * i) for i in range(few)] + [(70 + 9 * i, 200 + 50 * i) for i in range(many)], 16, dev, 23)
    p = Packed(b, d, bits, 8, 2, BF, dev, 440)
    check(p.run(), *p.reference())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 3, 2])
@pytest.mark.parametrize("lens", [[(4, 900), (1, 3000)], [(150, 900), (33, 400)]], ids=["few", "many"])
def test_float16_results_are_near_in_the_mean(dev, d, bits, lens):
    """Relative 2-norm of the error, with scores that spread by 4.  Roundings to float16 are 2^-10 / sqrt(12) at the lower end of a binade, 1.9e-4 of
    numbers spread over it: the result's own, the weights' (of terms as independent as the result's), and that of the
    levels, a quarter of it with the unit that suits them, times the 4 that scores are then off.  Together sqrt(3) x 1.9e-4 = 3.3e-4, where
    4.5e-4 is allowed; queries of one float16 term alone would add 4 x 1.9e-4."""
    p = Packed(Batch(lens, 16, dev, 24), d, bits, 8, 2, FP, dev, 450)
    levels = p.tq.centroids.double()
    spread = float((levels ** 2).mean().sqrt()) * math.sqrt(d) / 2 * math.sqrt(d) * p.attn.scale      # (norms are sqrt(d) / 2 in the middle)
    p.q = (p.q.double() * (4 / spread)).half()
    out, _ = p.reference()
    got = p.run().double()
    assert float((got - out).norm() / out.norm()) <= 4.5e-4
