"""What a scoring pass asks for: the rows that count (three parts of them, and of a piece of the weight, in fp32), a pair of numbers for every
token and 128 words (64 for up to 64 fp32 rows, which may run in narrower tiles), and a number a token.  (Sizes with enough tiles for whole ones.)"""
import pytest

from trimkv_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


SIZES = [(8192, 151936, 2048), (65536, 151936, 2048), (65, 50257, 768), (1500, 32000, 1001), (4096, 32000, 4096)]


@pytest.mark.parametrize("tokens,vocab,width,dtype", [(*s, d) for s in SIZES for d in ((0, 1) if s[0] == 4096 else (0, 1, 2))])
def test_scoring_asks_for_no_narrower_tiles_than_it_uses(lib, tokens, vocab, width, dtype):
    up = lambda n, to: -(-n // to) * to  # noqa: E731
    rows = up(tokens, 256)
    parts = 3 if dtype == 2 else 1
    piece = max(2048, (96 << 20) // (6 * width) // 256 * 256) if dtype == 2 else 0
    held = parts * 2 * width * (rows + up(piece, 256)) + tokens * 8 * (up(vocab, 128) // 128 + 2 * (vocab // max(piece, 1) + 2 if piece else 2))
    assert lib.tkv_vloss_workspace_bytes(tokens, vocab, width, dtype, 0, 0) <= held + 4 * tokens + (1 << 14)


@pytest.mark.parametrize("tokens", [1, 32, 33, 64])
def test_few_fp32_rows_have_room_for_narrow_tiles(lib, tokens):
    for width in (1, 8, 4096):
        assert lib.tkv_vloss_workspace_bytes(tokens, 100000, width, 2, 0, 0) >= 512 + 4 * tokens + tokens * 8 * -(-100000 // 64)
