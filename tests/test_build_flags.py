"""The build on a compiler that does not know an option of its insides."""
import pytest

from muserve_amd import build


def test_unknown_options_are_left_out(tmp_path, capfd):
    source, obj = tmp_path / "empty.hip", tmp_path / "empty.o"
    source.write_text("#include <hip/hip_runtime.h>\n__global__ void nothing() {}\n")
    build.compile_source(build.hipcc(), source, obj, ["-mllvm", "-no-such-option-at-all=1"])
    assert obj.stat().st_size > 0 and "built without" in capfd.readouterr().err


def test_errors_of_the_source_are_not(tmp_path):
    source = tmp_path / "wrong.hip"
    source.write_text("#include <hip/hip_runtime.h>\n__global__ void nothing() { no_such_thing(); }\n")
    with pytest.raises(RuntimeError, match="no_such_thing"):
        build.compile_source(build.hipcc(), source, tmp_path / "wrong.o", ["-mllvm", "-x-y-z=1"])


def test_the_options_are_known_here(tmp_path, capfd):
    source = tmp_path / "empty.hip"
    source.write_text("#include <hip/hip_runtime.h>\n__global__ void nothing() {}\n")
    for flags in build.EXTRA_FLAGS.values():
        build.compile_source(build.hipcc(), source, tmp_path / "empty.o", flags)
    assert "built without" not in capfd.readouterr().err
