"""Sizes that the launches of the operators for several position axes cannot count are refused when the graph is built."""
import pytest

MOST = (2 ** 32 - 1) // 256     # a workgroup of 256 threads a token, threads counted in 32 bits


@pytest.fixture
def ctx(pkg):
    c = pkg.Context()
    yield c
    c.free()


@pytest.mark.parametrize("n,streams,ok", [(MOST, 1, True), (MOST + 1, 1, False), (2 ** 23, 2, False), (2 ** 22, 3, True)])
def test_rope_tokens(ctx, n, streams, ok):
    x, pos = ctx.new_tensor("f16", 2, 1, n, streams), ctx.new_tensor("i32", 4 * n)
    for turn in (lambda: ctx.rope_multi(x, pos, None, 2, (1, 0, 0, 0), 8, 8192, 1e4), lambda: ctx.rope_multi_back(x, pos, None, 2, (1, 0, 0, 0), 8, 8192, 1e4),
                 lambda: ctx.rope_ext_back(x, ctx.new_tensor("i32", n), None, 2, 2, 8192, 1e4)):
        if ok:
            assert turn().ne == x.ne
        else:
            with pytest.raises(RuntimeError):
                turn()
