"""What the paged cache's binding decides on the host, without a device."""
import threading

import pytest

torch = pytest.importorskip("torch")


class Devices:
    """torch.cuda's view of two devices, the first current, `capturing` set for
    the current stream of the one whose index it names."""

    def __init__(self, monkeypatch, capturing):
        import whispereacp_b200.cache as module
        self.now, self.capturing = 0, capturing
        outer = self
        monkeypatch.setattr(module, "_workspaces", threading.local())

        class Guard:
            def __init__(self, index):
                self.index = index

            def __enter__(self):
                self.before, outer.now = outer.now, self.index

            def __exit__(self, *exc):
                outer.now = self.before
                return False

        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.now == self.capturing)


def cache_on(index):
    """A PagedCache as its workspaces see it, its memory the host's."""
    from whispereacp_b200 import PagedCache
    cache = PagedCache.__new__(PagedCache)
    cache._handle, cache._index, cache.device = None, index, torch.device("cpu")
    cache._raw_stream = lambda i: 1000 + i
    return cache


@pytest.mark.parametrize("index", [0, 1])
def test_a_captured_call_has_its_own_workspace_whichever_device_is_current(monkeypatch, index):
    devices = Devices(monkeypatch, capturing=index)
    cache = cache_on(index)
    first, second = cache._workspace(4096, None), cache._workspace(4096, None)
    assert first.data_ptr() != second.data_ptr()
    assert devices.now == 0


@pytest.mark.parametrize("index", [0, 1])
def test_a_call_beside_a_capture_on_another_device_shares_its_thread_s(monkeypatch, index):
    Devices(monkeypatch, capturing=1 - index)
    cache = cache_on(index)
    first, second = cache._workspace(4096, None), cache._workspace(2048, None)
    assert first.data_ptr() == second.data_ptr()
    assert cache_on(index)._workspace(4096, None).data_ptr() == first.data_ptr()


@pytest.mark.gpu
def test_waits_that_give_up(tmp_path):
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    program, library = os.path.join(str(tmp_path), "cache_wait_test"), os.path.join(root, "whispereacp_b200")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-ccbin", "g++",
                    "--expt-relaxed-constexpr", "-o", program, os.path.join(root, "tests", "cpp", "cache_wait_test.cu"),
                    "-L", library, "-lwsp_b200", "-Xlinker", f"-rpath={library}"], check=True)
    run = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
