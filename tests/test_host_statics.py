"""What the library's host code keeps between calls: host threads may call at once (ctypes
lets go of Python's lock), so a static variable is constant, atomic or locked."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "vllm-ascend-hust-latchmoe_amd" / "csrc"
SAFE = re.compile(r"static\s+(constexpr|const|std::atomic|LdsRaised|inline|__device__|void\* \(\*const)\b|static_assert|static_cast")


def test_statics_are_constant_or_atomic():
    found = []
    for path in sorted([*CSRC.glob("*.h"), *CSRC.glob("*.hip")]):
        for n, line in enumerate(path.read_text().splitlines(), 1):
            inner = re.match(r"\s+static\b", line)
            variable = re.match(r"\s+static\s[^(]*(=|;|\[)", line)
            if inner and variable and not SAFE.search(line):
                found.append(f"{path.name}:{n}: {line.strip()}")
    assert not found, "\n".join(found)


def test_raised_lds_is_atomic():
    assert "std::atomic<bool> on[64]" in (CSRC / "mx4_tile.h").read_text()
