"""The plugin is discoverable: pyproject.toml registers the engine in the `sklearn_engines`
entry-point group under the name `kmeans`, as the reference does (pyproject.toml:55-56 there),
and the registered object is the engine class with the protocol scikit-learn's engine API
calls."""
import importlib.metadata
import os
import subprocess
import sys
import tomllib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROTOCOL = ["accepts", "prepare_fit", "unshift_centers", "init_centroids", "kmeans_single",
            "is_same_clustering", "count_distinct_clusters", "prepare_prediction", "get_labels",
            "get_score", "prepare_transform", "get_euclidean_distances", "convert_to_sklearn_types"]


def _declared():
    with open(os.path.join(ROOT, "pyproject.toml"), "rb") as fh:
        return tomllib.load(fh)


def test_entry_point_is_declared_and_resolves_to_the_engine():
    meta = _declared()
    group = meta["project"]["entry-points"]["sklearn_engines"]
    assert list(group) == ["kmeans"]
    ep = importlib.metadata.EntryPoint(name="kmeans", value=group["kmeans"], group="sklearn_engines")
    engine_class = ep.load()
    from sklearn_numba_dpex_b200.kmeans.engine import KMeansEngine

    assert engine_class is KMeansEngine
    assert engine_class.engine_name == "kmeans"
    for method in PROTOCOL:
        assert callable(getattr(engine_class, method)), method
    # the provider name scikit-learn derives from the entry point's module
    assert ep.module.split(".")[0] == "sklearn_numba_dpex_b200"


def test_installed_distribution_exposes_the_same_entry_point():
    """When the distribution is installed (pip install -e . --no-build-isolation), discovery
    through importlib.metadata gives the same class; in a source checkout that was never
    installed there is nothing to look up and the declaration test above is the check."""
    found = [ep for ep in importlib.metadata.entry_points(group="sklearn_engines")
             if ep.value.startswith("sklearn_numba_dpex_b200.")]
    for ep in found:
        from sklearn_numba_dpex_b200.kmeans.engine import KMeansEngine

        assert ep.name == "kmeans" and ep.load() is KMeansEngine


def test_package_data_names_the_library_and_the_build_hook_exists():
    meta = _declared()
    assert "libkmb200.so" in meta["tool"]["setuptools"]["package-data"]["sklearn_numba_dpex_b200"]
    assert os.path.exists(os.path.join(ROOT, "setup.py"))
    assert os.path.exists(os.path.join(ROOT, "sklearn_numba_dpex_b200", "build.py"))


WITHOUT_CALLS = """
import sys
sys.modules["sklearn_numba_dpex_b200._torch_calls"] = None        # as if it were not built
import sklearn_numba_dpex_b200.kmeans.drivers
from sklearn_numba_dpex_b200.common.random import create_xoroshiro128pp_states
from sklearn_numba_dpex_b200.common import get_random_raw, topk, topk_idx
from sklearn_numba_dpex_b200 import common
assert callable(topk) and callable(topk_idx) and callable(common.topk)
assert {"topk", "route_topk", "int8_matmul"} <= set(dir(common))
assert not hasattr(common, "no_such_helper")
for name in ("route_topk", "int8_matmul", "experts", "int8"):
    try:
        getattr(common, name)
    except ImportError as exc:
        assert "sklearn_numba_dpex_b200.build" in str(exc), exc
    else:
        raise SystemExit(name + " did not miss its extension")
print("without-ok")
"""


def test_engine_and_helpers_need_no_extension():
    """A fit with k-means++ seeding, top-k and the random helpers work without the extension of the expert calls;
    those name the command that builds it."""
    proc = subprocess.run([sys.executable, "-c", WITHOUT_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0 and "without-ok" in proc.stdout, proc.stdout + proc.stderr


def test_names_of_the_helpers_are_what_their_modules_hold():
    from sklearn_numba_dpex_b200 import common
    from sklearn_numba_dpex_b200.common import experts, int8

    for module, names in ((experts, ("route_topk", "route_topk_grad", "expert_slots", "combine_experts", "combine_experts_grad")),
                          (int8, ("quantize_rows", "int8_matmul", "check_int8_waits"))):
        for name in names:
            assert getattr(common, name) is getattr(module, name)
    held = {}
    exec("from sklearn_numba_dpex_b200.common import *", held)
    assert set(common.__all__) <= set(held)


def test_extension_of_another_torch_or_interpreter_is_built_anew(tmp_path, monkeypatch):
    """By what it was built for, not by the time of its file alone: an extension that is newer than every source
    is kept for the same torch, and built again for another one."""
    import torch

    from sklearn_numba_dpex_b200 import build

    compiled = []

    def compiler(cmd, **kw):
        compiled.append(cmd)
        (tmp_path / "_torch_calls.so").write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "CALLS_PATH", str(tmp_path / "_torch_calls.so"))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(build, "CALLS_STAMP", str(tmp_path / "torch_calls.stamp"), raising=False)
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_calls()
    build.build_calls()
    assert len(compiled) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_calls()
    build.build_calls()
    assert len(compiled) == 2 and any("9.9.9" in word for word in compiled[1])
    monkeypatch.setattr(build.sys, "version", "9.9")
    build.build_calls()
    assert len(compiled) == 3
    (tmp_path / "_torch_calls.so").unlink()
    build.build_calls()
    assert len(compiled) == 4


OTHER_TORCH = """
import torch
torch.__version__ = "9.9.9"
from sklearn_numba_dpex_b200 import common
try:
    common.route_topk
except ImportError as exc:
    assert "built for torch" in str(exc) and "9.9.9" in str(exc) and "sklearn_numba_dpex_b200.build" in str(exc), exc
    print("refused-ok")
"""


def test_extension_of_another_torch_is_refused():
    proc = subprocess.run([sys.executable, "-c", OTHER_TORCH], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0 and "refused-ok" in proc.stdout, proc.stdout + proc.stderr


def test_build_without_torch_leaves_the_extension_out(tmp_path, monkeypatch, capsys):
    """torch is no build requirement, which pip would fetch in a version of its own: an isolated build ships the
    library and says how to get the rest."""
    from sklearn_numba_dpex_b200 import build

    assert not any(r.startswith("torch") for r in _declared()["build-system"]["requires"])
    (tmp_path / "lib.so").write_bytes(b"")
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "_nvcc", lambda: "nvcc")
    monkeypatch.setattr(build, "_compile_one", lambda nvcc, src, force, verbose: (str(tmp_path / "lib.so"), ""))
    calls = []
    monkeypatch.setattr(build, "build_calls", calls.append)
    assert build.build() == str(tmp_path / "lib.so") and calls == [False]
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build.build() == str(tmp_path / "lib.so") and calls == [False]
    assert "--no-build-isolation" in capsys.readouterr().out
