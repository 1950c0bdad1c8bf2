"""What makes an object out of date."""
import importlib.util
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_an_object_is_built_again_when_its_flags_change(monkeypatch):
    """the flags of each source are in build.py: an object that is older was compiled with others"""
    path = os.path.join(ROOT, "coco-dr_amd", "build.py")
    spec = importlib.util.spec_from_file_location("_build_under_test", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    asked = {}
    monkeypatch.setattr(mod, "_stale", lambda out, deps: asked.update({os.path.basename(out): [os.path.basename(d) for d in deps]}) or False)
    mod.build_library()
    for s in mod.SOURCES:
        deps = asked[s.replace(".hip", ".o")]
        assert s in deps and "cocodr.h" in deps and "build.py" in deps, s
