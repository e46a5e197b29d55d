"""Write ``docs/python_api.md``: the public surface of the package with signatures and the first
paragraph of every docstring.

    python docs/gen_api.py            # rewrites docs/python_api.md
    python docs/gen_api.py --check    # exit 1 if the committed page is out of date

Parity: the ``docs/source/python_api`` pages of the reference (Sphinx autodoc there).
"""
from __future__ import annotations

import importlib
import inspect
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(HERE))

SECTIONS = [
    ("Schedule language", "slapo_b200", ["create_schedule", "build", "Verify", "init_empty_weights",
                                         "set_random_seed", "get_cuda_rng_tracker", "list_primitives"]),
    ("Schedule object", "slapo_b200.schedule", ["Schedule"]),
    ("Patterns", "slapo_b200.pattern", ["Pattern", "ModulePattern", "call_module"]),
    ("Model schedules", "slapo_b200.model_schedule", ["apply_schedule", "register_schedule",
                                                      "list_schedules"]),
    ("Ops", "slapo_b200.op", None),
    ("Functional kernels", "slapo_b200.ops.functional", ["linear", "linear_t", "gemm", "bias_act",
                                                         "dropout_add_layer_norm", "flash_attention",
                                                         "embedding", "rotary", "rotary_qkvpacked",
                                                         "paged_append", "paged_attention", "sample",
                                                         "effective_dropout_p"]),
    ("Tensor-parallel fused ops", "slapo_b200.parallel.fused_tp",
     ["ag_linear", "rs_linear", "ar_linear", "ag_gemm", "ag_gemm_pushed", "gemm_rs", "gemm_ar",
      "peer_gather", "ag_mode", "StagePool"]),
    ("Mesh and symmetric memory", "slapo_b200.parallel.mesh", ["DeviceMesh"]),
    ("Symmetric memory", "slapo_b200.parallel.symm", ["SymmContext", "SymmBuffer"]),
    ("Sharding solver", "slapo_b200.parallel.solver", ["solve_sharding"]),
    ("Engines", "slapo_b200.runtime.engine", ["TrainEngine", "EngineConfig"]),
    ("Pipeline engine", "slapo_b200.runtime.pipeline_engine", ["PipelineEngine"]),
    ("Failure detection", "slapo_b200.runtime.health", None),
    ("Checkpoints", "slapo_b200.ckpt", ["save_checkpoint", "load_checkpoint",
                                        "consolidate_checkpoint", "reshard_checkpoint"]),
    ("Data", "slapo_b200.data", ["pack_documents", "TokenFileDataset", "SyntheticDataset",
                                 "build_dataloader", "DevicePrefetcher"]),
    ("Auto-tuner", "slapo_b200.autotune.tune", ["Symbol", "Space", "Database", "tune"]),
    ("Utilities", "slapo_b200.utils.report", None),
]


def first_paragraph(obj):
    doc = inspect.getdoc(obj) or ""
    para = doc.split("\n\n")[0].strip()
    return " ".join(line.strip() for line in para.splitlines())


def signature(obj):
    try:
        return str(inspect.signature(obj))
    except (TypeError, ValueError):
        return "(...)"


def public_names(mod):
    names = getattr(mod, "__all__", None)
    if names is None:
        names = [n for n, o in vars(mod).items()
                 if not n.startswith("_") and (inspect.isclass(o) or inspect.isfunction(o))
                 and getattr(o, "__module__", "").startswith("slapo_b200")]
    return sorted(names)


def render():
    out = ["# Python API", "",
           "Generated by `python docs/gen_api.py` from the docstrings; do not edit by hand.", ""]
    for title, modname, names in SECTIONS:
        mod = importlib.import_module(modname)
        out += [f"## {title} (`{modname}`)", ""]
        for name in names if names is not None else public_names(mod):
            obj = getattr(mod, name, None)
            if obj is None:
                continue
            kind = "class" if inspect.isclass(obj) else "def"
            out.append(f"### `{kind} {name}{signature(obj)}`")
            para = first_paragraph(obj)
            if para:
                out += ["", para]
            if inspect.isclass(obj):
                wrappers = (staticmethod, classmethod)
                methods = [(n, m) for n, m in vars(obj).items() if not n.startswith("_")
                           and (inspect.isfunction(m) or isinstance(m, wrappers))]
                for n, m in methods:
                    fn = m.__func__ if isinstance(m, (staticmethod, classmethod)) else m
                    line = f"* `{n}{signature(fn)}`"
                    para = first_paragraph(fn)
                    out.append(line + (f" - {para}" if para else ""))
            out.append("")
    return "\n".join(out).rstrip() + "\n"


def main(argv):
    path = os.path.join(HERE, "python_api.md")
    text = render()
    if "--check" in argv:
        with open(path, encoding="utf-8") as fh:
            return 0 if fh.read() == text else 1
    with open(path, "w", encoding="utf-8") as fh:
        fh.write(text)
    print(path, f"{len(text.splitlines())} lines")
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
