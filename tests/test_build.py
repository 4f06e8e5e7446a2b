"""The build command."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_c_library_builds_without_torch():
    """A host of the C ABI alone has no torch."""
    code = ("import runpy, sys; sys.modules['torch'] = None; sys.argv = ['build.py']; "
            f"runpy.run_path({os.path.join(ROOT, 'rapidocrvl_b200', 'build.py')!r}, run_name='__main__')")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "libocrvl_cuda.so" in r.stdout and "not built" in r.stdout
