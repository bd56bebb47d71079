"""The record of measured memory traffic that bench.py quotes lies in the tree that runs on the GPU."""
import json
import os
import re

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_the_traffic_record_is_there():
    names = re.findall(r'"((?:r\d_)?pmc_traffic\.json)"', open(os.path.join(ROOT, "bench.py")).read())
    there = [n for n in names if os.path.exists(os.path.join(ROOT, "profiles", n))]
    assert names and there and there[0] == names[0]
    record = json.load(open(os.path.join(ROOT, "profiles", there[0])))
    assert any("hbm_bytes_corrected" in r and "algorithmic_bytes" in r and "shape" in r for r in record.values() if isinstance(r, dict))
