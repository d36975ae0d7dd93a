"""The device's error slot is shared by all streams and threads: nothing but an atomic writes it."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "greyhound_b200" / "csrc"


def test_error_slots_are_written_by_one_atomic():
    sources = {p.name: re.sub(r"//.*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu*"))}
    # a load, an OR and a store through one pointer
    plain = re.compile(r"\*\s*(\w+)\s*(?:=\s*\*\s*\1\s*\||\|=)")
    assert [(n, m.group(0)) for n, s in sources.items() for m in plain.finditer(s)] == []
    assert "atomicOr(slot, bits)" in sources["common.cuh"]
    for name in ("capi.cu", "lsm.cu", "token_losses.cu"):
        assert "report_bits(" in sources[name]
        assert not re.search(r"\bslot\s*=\s*[*(]|\*\s*(?:q\.)?slot\s*=\s*[^n=]*\|", sources[name])
