"""The build recipe (candle-fused-attn_amd/build.py), without a GPU."""
from __future__ import annotations

import importlib.util
from pathlib import Path

RECIPE = Path(__file__).resolve().parent.parent / "candle-fused-attn_amd" / "build.py"


def test_builds_are_reproducible(tmp_path):
    """The same source compiled in two folders, as two builds do, is the same file: profiles/traffic.json
    holds for a library by its hash."""
    spec = importlib.util.spec_from_file_location("fattn_build_recipe", RECIPE)
    recipe = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(recipe)
    built = []
    for name in ("a", "b"):
        (tmp_path / name).mkdir()
        (out,) = recipe.compile_objects([recipe.CSRC / "fattn_operators.cpp"], tmp_path / name)
        built.append(out.read_bytes())
    assert built[0] == built[1]
