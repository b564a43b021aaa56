"""What makes the built libraries out of date (no GPU needed)."""

from purin_b200.csrc import build


def test_binding_of_another_torch_is_out_of_date(tmp_path, monkeypatch):
    if not build.up_to_date():
        build.build()
    assert build.up_to_date()
    for text in ("torch 1.0, cpython-312\n", None):
        stamp = tmp_path / "built_for"
        if text is not None:
            stamp.write_text(text)
        else:
            stamp.unlink()
        monkeypatch.setattr(build, "TORCH_STAMP", stamp)
        assert not build.up_to_date()
    monkeypatch.undo()
    assert build.up_to_date()
