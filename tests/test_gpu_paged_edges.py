"""The serving operators where several of their rules meet: chunks that pass the end of their table.  Against plain 64-bit forms
on the CPU (``paged_reference``)."""
import math
import sys

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _ops():
    from mindpipe_amd import ops
    return ops


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- chunks that pass the end of their table
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,grp,width", [(64, 7, 5), (128, 1, 5), (256, 4, 5), (128, 2, 60), (256, 1, 60)])
@pytest.mark.parametrize("bad", [False, True])
def test_chunks_past_the_end_of_their_table(dtype, dim, grp, width, bad):
    """A row sees the positions up to the one that the append gives it, as far as the table goes: also where the sequence's
    length passes the table's room and the last rows of the chunk have no place.  Wide tables split their positions.  ``bad``: an
    infinity in a value that only some of the rows see, whose rows are done again."""
    kvh, page = 2, 16
    room = width * page
    news = [4, 40, 9, 3, 5, 2]
    lens = [room + 2, room + 39, room, room - 1, room + 5000, 2 ** 31 - 1]
    _say("chunks past the table", dtype, dim, grp, width, bad)
    g = torch.Generator().manual_seed(dim + width)
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    pages = len(lens) * width
    k, v = (torch.randn(pages, kvh, page, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    table = torch.randperm(pages, generator=g).view(len(lens), width).to(torch.int32)
    nh = kvh * grp
    qkv = torch.randn(at[-1], (nh + 2 * kvh) * dim, generator=g).to(dtype).to(DEV)
    angle = torch.rand(room + 50, dim // 2, generator=g) * 6.3
    q = _ops().paged_rope_append(qkv, angle.cos().to(DEV), angle.sin().to(DEV), k, v, table.to(DEV), _ints(lens), _ints(at))
    q = torch.randn(q.shape, generator=g).to(dtype).to(DEV)  # (positions without an angle have zero queries)
    # which position each row has is the append's to say: the new keys are where it put them
    x, cos, sin = qkv.cpu().view(at[-1], -1, dim), angle.cos(), angle.sin()
    kc, vc = k.cpu(), v.cpu()
    for b, n in enumerate(news):
        for j in range(n):
            pos = lens[b] - n + j
            if pos >= room:
                continue
            page_of, row = int(table[b, pos // page]), pos % page
            assert torch.equal(vc[page_of, :, row], x[at[b] + j, nh + kvh:])
            want = ref.rotate(x[at[b] + j:at[b] + j + 1, nh:nh + kvh].double(), cos[pos:pos + 1], sin[pos:pos + 1], True)[0]
            assert ((kc[page_of, :, row].double() - want).abs() <= ref.HALF_STEP[dtype] * want.abs() + 2.0 ** -20).all()
    if bad:  # the table's last position of the first two sequences: the first row of the first chunk does not see it
        for b in (0, 1):
            v[int(table[b, -1]), 0, page - 1] = math.inf
        vc = v.cpu()
    got = _ops().paged_prompt_attention(q, k, v, table.to(DEV), _ints(lens), _ints(at), dim ** -0.5)
    qc = q.cpu().double()
    for b, n in enumerate(news):
        rows_k, rows_v = (t[table[b].long()].transpose(1, 2).reshape(room, kvh, dim).double() for t in (kc, vc))
        for j in range(n):
            sees = min(lens[b] - n + j + 1, room)
            for h in range(nh):
                want, bound = ref.attention_row(qc[at[b] + j, h], rows_k[:sees, h // grp], rows_v[:sees, h // grp], dim ** -0.5)
                if torch.isfinite(want).all():
                    ref.check(got[at[b] + j, h], want, ref.allowed(bound, dtype), what=f"sequence {b} row {j} head {h}")
                else:
                    assert not torch.isfinite(got[at[b] + j, h]).any()
