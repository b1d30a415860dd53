"""What the scores' statistics need of the workspace: bounded, whatever the tokens are, and enough for each run of them.  No GPU needed."""
import pytest

from loss_choice import score_run

TOKENS = [1, 64, 65, 255, 256, 257, 1000, 2049, 4096, 5001, 16384, 16385, 20000, 70001, 131072, 1 << 20, (1 << 26) - 1, 1 << 26]


@pytest.mark.parametrize("vocabulary", [1, 5000, 32003, 128256, 262145, 1 << 21, 1 << 26])
def test_statistics_are_bounded(miw, vocabulary):
    """128 MiB, or those of 256 tokens, beside what a token has for itself."""
    for tokens in TOKENS:
        need = miw.LOSS.cross_entropy_workspace(tokens, vocabulary, 64)
        assert need <= 8 * max(1 << 24, 256 * (-(-vocabulary // 32) + 8), 64 * (-(-vocabulary // 16) + 8)) + 8 * tokens + 512, tokens


@pytest.mark.parametrize("vocabulary", [1, 5000, 32003, 128256, 262145, 1 << 21, 1 << 26])
@pytest.mark.parametrize("width,vector", [(8, True), (64, True), (2048, True), (65, False)])
def test_each_run_has_room(miw, vocabulary, width, vector):
    for tokens in TOKENS:
        run, slices = score_run(miw, tokens, vocabulary, width, vector)
        assert 1 <= run <= tokens and (run == tokens or run % 256 == 0)
        assert 8 * run * slices + 8 * run <= miw.LOSS.cross_entropy_workspace(tokens, vocabulary, width), (tokens, run, slices)
        # tokens in one run where there is room for it
        assert run == tokens or 8 * tokens * slices > 1 << 27 or run * 2 > tokens, (tokens, run, slices)
    assert score_run(miw, 16384, 128256, 2048)[0] == 16384


@pytest.mark.parametrize("vocabulary,width", [(1, 1), (5000, 64), (32003, 2048), (128256, 8), (128256, 2048), (1 << 21, 64)])
@pytest.mark.parametrize("piece", [0, 1, 1000])
def test_a_gradients_workspace_does_for_the_scores(miw, vocabulary, width, piece):
    for tokens in TOKENS:
        assert miw.LOSS.cross_entropy_workspace(tokens, vocabulary, width, grad=True, piece=piece) >= miw.LOSS.cross_entropy_workspace(tokens, vocabulary, width), tokens
