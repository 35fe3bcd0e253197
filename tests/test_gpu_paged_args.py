"""Arguments that the JavaScript API of the paged cache and of verifyDrafts refuses
(tests/js/paged_args.mjs)."""
import json
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_refused_arguments(fh):
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "paged_args.mjs")], stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, env=dict(os.environ, FORGE_DEVICE="0"), timeout=100)
    lines = [json.loads(x) for x in r.stdout.splitlines() if x.startswith("{")]
    assert lines and all(x["ok"] for x in lines) and r.returncode == 0, r.stdout
