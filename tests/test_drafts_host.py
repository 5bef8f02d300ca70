"""The draft look-up of the greedy loop (arbolDe), on the CPU: shapes, limits and the order of the tree's tokens."""
import json
import os
import subprocess

import pytest

from conftest import ROOT

TF = os.path.join(ROOT, "quipullm_amd", "js", "transformer.js")


def tree(h, most, deep):
    s = ("const {arbolDe} = require(%s); const a = arbolDe(%s, %d, %d); console.log(JSON.stringify("
         "{ids: a.ids, padres: a.padres, hijos: a.ids.map((x, i) => a.ids.map((y) => a.hijo(i, y)))}));")
    out = subprocess.run(["node", "-e", s % (json.dumps(TF), json.dumps(h), most, deep)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    return json.loads(out.stdout)


def test_no_earlier_occurrence():
    assert tree([1, 2, 3], 16, 8)["ids"] == [3]
    assert tree([5], 16, 8) == {"ids": [5], "padres": [-1], "hijos": [[-1]]}


def test_longest_match_first_and_shared_prefixes():
    #  1 2 3 4 5 | 9 1 2 3 4 6 | 0 1 2 3: after (1, 2, 3) came 4 6 (later) and 4 5 (earlier)
    a = tree([1, 2, 3, 4, 5, 9, 1, 2, 3, 4, 6, 0, 1, 2, 3], 16, 3)
    assert a["ids"][0] == 3 and a["padres"][0] == -1
    ways = set()
    for i in range(len(a["ids"])):
        way, j = [], i
        while j >= 0:
            way.insert(0, a["ids"][j])
            j = a["padres"][j]
        ways.add(tuple(way))
    assert ways == {(3,), (3, 4), (3, 4, 6), (3, 4, 5)}
    assert all(p < i for i, p in enumerate(a["padres"]))
    assert a["hijos"][0][1] == 1 and a["hijos"][1][0] == -1


@pytest.mark.parametrize("most", [1, 2, 5, 16])
@pytest.mark.parametrize("deep", [1, 2, 7])
def test_limits(most, deep):
    """At most `most` tokens, none deeper than deep - 1 below the root (deep tokens are still wanted, the model's own choice
    behind the path among them)."""
    a = tree([1, 2, 3, 1, 2, 4, 1, 2, 5, 1, 2], most, deep)
    assert 1 <= len(a["ids"]) <= most
    for i in range(len(a["ids"])):
        d, j = 0, i
        while a["padres"][j] >= 0:
            d, j = d + 1, a["padres"][j]
        assert d <= deep - 1


@pytest.mark.parametrize("most", [1.5, 2.5, 4.25])
def test_limits_that_are_no_whole_numbers(most):
    """A tree stays below the limit, whole or not."""
    s = ("const {arbolDe} = require(%s); console.log(arbolDe(%s, %s, 9).ids.length);"
         % (json.dumps(TF), json.dumps([1, 2, 3, 4, 5, 6, 7, 8, 9, 1, 2]), most))
    out = subprocess.run(["node", "-e", s], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    assert int(out.stdout) <= most
