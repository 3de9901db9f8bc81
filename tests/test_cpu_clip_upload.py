"""apexw_clip_upload's refusals: nothing is launched."""

from apexw_amd import _lib


def test_refusals():
    upload, ok = _lib.load().apexw_clip_upload, 4096
    assert upload(None, 1, ok, None) == 1 and upload(ok, 1, None, None) == 1 and upload(ok, -1, ok, None) == 1
    assert upload(ok, 1, ok + 4, None) == 4
    assert upload(None, 0, None, None) == 0
