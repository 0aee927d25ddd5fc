"""Every stream of this repository has the default priority: a fresh high-priority stream that waits for a busy one has been
seen never to drain."""
import re
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
SOURCES = [p for d in ("d-vqvae_amd", "tools", "tests", "oracle", "perf", "include") for p in sorted((ROOT / d).rglob("*"))
           if p.suffix in (".py", ".hip", ".h", ".cpp", ".sh") and p != Path(__file__).resolve()] + [ROOT / "bench.py"]
OTHER_PRIORITY = re.compile(r"Stream\([^)\n]*priority|StreamCreateWithPriority|is_high_priority_stream\s*=\s*True")


def test_no_source_makes_a_stream_of_another_priority():
    assert len(SOURCES) > 50
    found = [f"{p.relative_to(ROOT)}:{i}" for p in SOURCES for i, line in enumerate(p.read_text(errors="replace").splitlines(), 1)
             if OTHER_PRIORITY.search(line)]
    assert not found, found
