"""Document ids of laya_b200_attention_varlen: any negative id marks a key that nobody sees and a query that
sees nothing, whichever negative number it is. Checked against the formula in 64 bits with the bounds of the
attention tests."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_attention_varlen_gpu import gpu, run  # noqa: E402, F401

NEGATIVE = [-1, -2, -3, -4, -(2 ** 31)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("negative", NEGATIVE + [0])
def test_negative_ids_in_mixed_chunks(D, negative):
    """Keys and queries of one negative id (0: of all of them) among keys of the rows' documents."""
    rng = random.Random(negative)
    pick = lambda: rng.choice(NEGATIVE) if negative == 0 else negative  # noqa: E731
    lens = [200, 64, 513]
    ids = [[pick() if rng.random() < 0.3 else rng.choice([0, 1]) for _ in range(n)] for n in lens]
    out, lse = run(lens, D=D, docs=(ids, ids))
    dead = torch.tensor(sum(ids, []), device="cuda") < 0
    n = sum(lens)
    assert bool((lse[:n][dead] == -math.inf).all()) and bool((out[:n][dead] == 0).all())
    other = [[pick() if rng.random() < 0.5 else 1 for _ in range(n)] for n in lens]
    run(lens, D=D, docs=(other, ids), right=0, cap=20.0)
    run([1, 2, 1], [300, 70, 5], D=D, Hq=8, Hkv=2,
        docs=([[pick()], [0, pick()], [1]], [x[:n] for x, n in zip([ids[2], ids[0], ids[1]], [300, 70, 5])]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("negative", [-2, -3, -4])
def test_negative_ids_past_the_document_map(D, negative):
    """Whole chunks of a negative id behind the first 4096 chunks, for rows of several documents."""
    lk = 4096 * 64 + 64 * 12
    kd = [i // 30000 for i in range(lk)]
    for c in (2, 3, 7, 11):
        at = (4096 + c) * 64
        kd[at:at + 64] = [negative] * 64
    run([100], [lk], D=D, Hq=1, Hkv=1, docs=([[8] * 40 + [negative] * 10 + [7] * 50], [kd]))
    run([3], [lk], D=D, Hq=1, Hkv=1, docs=([[8, negative, 7]], [kd]))
