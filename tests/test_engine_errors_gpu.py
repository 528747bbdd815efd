"""GPU test of an engine that does not fit the card: the error is that call's alone."""
import pytest

pytestmark = pytest.mark.gpu


def test_engine_after_one_that_does_not_fit(cuda):
    """The allocation of an engine larger than the card fails; the next engine loads and runs as before."""
    from strataflow_b200 import engine as E
    from strataflow_b200 import lib as L
    cfg = E.tiny_config(n_layer=1, n_ctx=16)
    want = E.Engine.load(cfg, seed=0).forward(1, 0)[0]
    with pytest.raises(L.SfkError) as e:
        E.Engine(E.tiny_config(n_vocab=800_000_000))
    assert e.value.status == L.SFK_ERR_OUT_OF_MEMORY
    eng = E.Engine.load(cfg, seed=0)
    assert eng.forward(1, 0)[0] == want
