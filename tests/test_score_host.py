"""Host checks of the scoring model (auratensor_b200/score.py): what they refuse reaches neither the cache nor a GPU."""
import pytest

from auratensor_b200 import _lib
from auratensor_b200.inference import LlamaConfig
from auratensor_b200.score import BlockLlama, main
from auratensor_b200.synth import TINY


class Untouched:
    def __getattr__(self, name):
        raise AssertionError(f"the cache was asked for {name}")


def model():
    m = BlockLlama.__new__(BlockLlama)
    m.config, m.cache = LlamaConfig.fromShape(TINY), Untouched()
    return m


@pytest.mark.parametrize("ids", [[TINY.vocab], [1, 2, TINY.vocab + 5], [-1], [3, -2, 4], [1 << 40]])
def test_token_ids_outside_the_vocabulary_are_refused(ids):
    for call in (lambda: model().forward([(0, 0, ids)]), lambda: model().forward([(0, 0, [1]), (1, 0, ids)])):
        with pytest.raises(_lib.IllegalArgumentException, match="out of range"):
            call()


@pytest.mark.parametrize("start,n", [(TINY.ctx, 1), (TINY.ctx - 3, 4), (0, TINY.ctx + 1), (1 << 40, 1)])
def test_positions_past_the_context_are_refused(start, n):
    """The cache's last block may end past the context: the rotary table does not."""
    with pytest.raises(_lib.IllegalStateException, match="exceeds maxContext"):
        model().forward([(0, start, [1] * n)])
    with pytest.raises(_lib.IllegalArgumentException, match="negative"):
        model().forward([(0, -1, [1])])


@pytest.mark.parametrize("args", [["--ids", "5"], ["--ids", ""], ["--texts", "0"], ["--texts", "-1"]])
def test_a_command_with_nothing_to_score_is_refused(args, capsys):
    with pytest.raises(SystemExit) as e:
        main(args)
    assert e.value.code == 2 and "at least" in capsys.readouterr().err


def test_no_texts_have_no_scores():
    assert model().score([]) == []
