"""The decode example notices a step whose sequences did not get the pages that they asked for."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def load():
    path = Path(__file__).resolve().parent.parent / "examples" / "kv_decode.py"
    spec = importlib.util.spec_from_file_location("kv_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("short", [None, 0, 3, 4])
def test_steps_without_pages_are_noticed(short):
    """`short`: the step in which one sequence gets no page; 80 + 5 tokens, so a block begins with the
    first step and the other steps go on in it."""
    module = load()
    resize, calls = module.kv_resize, []

    def less(refs, table, lengths, want, **kw):
        got = resize(refs, table, lengths, want, **kw)
        calls.append(got)
        if short is not None and len(calls) == 2 + short:  # behind the prompt's call
            limits = got.limits.clone()
            limits[1] = lengths[1]
            got = got._replace(limits=limits)
        return got

    module.kv_resize = less
    run = lambda: module.run(seqs=2, context=80, steps=5, top=3, keep=9, q_heads=8, kv_heads=2)  # noqa: E731
    if short is None:
        assert run()["steps"] == 5
    else:
        with pytest.raises(AssertionError):
            run()
    assert len(calls) == 6
