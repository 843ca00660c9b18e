"""flashinfer-bench solution packaging of the B200 GDN operators.

The reference packs each operator as a flashinfer-bench *solution*: a JSON dict
with name, definition, author, a build spec and the source files
(gdn/benchmarks/bench_modal.py:99-144, gdn/decode/scripts/pack_solution.py:17-50).
``build_solution_dict(op)`` produces the same structure for this package with
``language = "cuda"``: the sources are the CUDA files, the C-ABI header and the
Python host modules, plus a generated entry file ``kernel.py`` whose ``kernel``
is this package's operator. On first import in the harness the entry compiles
the library from the bundled sources with nvcc (sm_100a) next to them.
"""
from __future__ import annotations

import json
from pathlib import Path

PKG = "flashinfer_bench_tma_thrust_b200"
PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent

SOLUTIONS = {
    "decode": {"name": "b200-gdn-decode", "definition": "gdn_decode_qk4_v8_d128_k_last",
               "module": "decode"},
    "prefill": {"name": "b200-gdn-prefill-chunked", "definition": "gdn_prefill_qk4_v8_d128_k_last",
                "module": "prefill"},
}
AUTHOR = "gdn-b200"
ENTRY = "kernel.py::kernel"
HOST_MODULES = ("__init__.py", "_lib.py", "_checks.py", "_status.py", "build.py", "decode.py",
                "prefill.py", "short_conv.py", "ssm.py", "partition.py", "workloads.py")

ENTRY_TEMPLATE = '''"""Entry point of the {name} solution (generated by {pkg}.solution)."""
import os
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
if _HERE not in sys.path:
    sys.path.insert(0, _HERE)

from {pkg} import build as _build  # noqa: E402

_build.build()
from {pkg}.{module} import kernel  # noqa: E402,F401
'''


def source_files() -> list[tuple[str, Path]]:
    """(relative path inside the solution, file on disk) of every bundled source."""
    out = []
    for name in HOST_MODULES:
        out.append((f"{PKG}/{name}", PKG_DIR / name))
    for f in sorted((PKG_DIR / "csrc").iterdir()):
        if f.suffix in (".cu", ".cuh", ".h"):
            out.append((f"{PKG}/csrc/{f.name}", f))
    for f in sorted((REPO_DIR / "include").glob("*.h")):
        out.append((f"include/{f.name}", f))
    return out


def build_solution_dict(op: str) -> dict:
    cfg = SOLUTIONS[op]
    sources = [{"path": "kernel.py",
                "content": ENTRY_TEMPLATE.format(name=cfg["name"], pkg=PKG, module=cfg["module"])}]
    sources += [{"path": rel, "content": f.read_text()} for rel, f in source_files()]
    return {
        "name": cfg["name"],
        "definition": cfg["definition"],
        "author": AUTHOR,
        "spec": {
            "language": "cuda",
            "target_hardware": ["cuda"],
            "entry_point": ENTRY,
            "dependencies": [],
            "destination_passing_style": False,
        },
        "sources": sources,
    }


def write_solution(op: str, path) -> Path:
    path = Path(path)
    path.write_text(json.dumps(build_solution_dict(op), indent=2))
    return path


def materialize(solution: dict, directory) -> Path:
    """Write a solution's sources into `directory` (what a harness does before import)."""
    d = Path(directory)
    for s in solution["sources"]:
        f = d / s["path"]
        f.parent.mkdir(parents=True, exist_ok=True)
        f.write_text(s["content"])
    return d


if __name__ == "__main__":
    import argparse

    ap = argparse.ArgumentParser(description="write a flashinfer-bench solution JSON")
    ap.add_argument("op", choices=sorted(SOLUTIONS))
    ap.add_argument("out")
    a = ap.parse_args()
    print(write_solution(a.op, a.out))
