"""What __graft_entry__.smoke() does where the plugin is not built."""
import pytest

import __graft_entry__ as entry
import llamacog_amd as la
from llamacog_amd import gguf_synth


@pytest.fixture
def unbuilt(monkeypatch, tmp_path):
    """No plugin, no host stack, no headers; the operators' part left out.  Returns the headers' root."""
    monkeypatch.setattr(entry, "_smoke_device_ops", lambda: None)
    monkeypatch.setattr(entry, "REF", str(tmp_path / "ref"))
    monkeypatch.setattr(la, "PLUGIN", str(tmp_path / "libggml-mi355x.so"))
    monkeypatch.setattr(la, "LLB", str(tmp_path / "libllb.so"))
    monkeypatch.setattr(la, "REFHOST", str(tmp_path))
    monkeypatch.setattr(gguf_synth, "ensure", lambda name: name)
    return tmp_path / "ref"


def test_smoke_without_headers_runs_the_operators_alone(unbuilt, capsys):
    entry.smoke()
    assert "operators alone" in capsys.readouterr().out


def test_smoke_fails_where_the_plugin_could_have_been_built(unbuilt):
    include = unbuilt / "ggml" / "include"
    include.mkdir(parents=True)
    (include / "ggml.h").touch()
    with pytest.raises(la.BackendMissing):
        entry.smoke()
