"""Which engine a runtime gets for its options (no GPU: loading is replaced by a record of what was asked for)."""
import pytest

from speech_to_text_amd.runtimes import mi355x_runtime as M


@pytest.fixture
def loads(monkeypatch):
    made = []

    def load(path, *, gelu=None, decoder_format='bf16', encoder_mlp_format='bf16', **kwargs):
        e = M._Engine({'n_vocab': 7}, {}, gelu_tanh=gelu in (None, 'tanh'),
                      formats=dict(decoder_format=decoder_format, encoder_mlp_format=encoder_mlp_format))
        made.append((path, gelu, decoder_format, encoder_mlp_format))
        return e
    monkeypatch.setattr(M.MI355XRuntime, 'load_engine', staticmethod(load))
    monkeypatch.setattr(M.MI355XRuntime, '_engines', {})
    monkeypatch.setattr(M.MI355XRuntime, '_format_engines', {})
    return made


@pytest.mark.parametrize('formats', [{}, dict(decoder_format='mxfp4'), dict(decoder_format='mxfp4', encoder_mlp_format='mxfp4')])
def test_each_form_of_gelu_has_its_engine(loads, formats):
    plain = M.MI355XRuntime('p', **formats)
    erf = M.MI355XRuntime('p', gelu='erf', **formats)
    tanh = M.MI355XRuntime('p', gelu='tanh', **formats)
    assert plain.engine.gelu_tanh and tanh.engine is plain.engine
    assert not erf.engine.gelu_tanh and erf.engine is not plain.engine
    assert M.MI355XRuntime('p', gelu='erf', **formats).engine is erf.engine
    assert M.MI355XRuntime('p', **formats).engine is plain.engine
    assert len(loads) == 2
    for r in (plain, erf):
        assert {k: r.engine.formats[k] for k in formats} == formats
    with pytest.raises(ValueError):
        M.MI355XRuntime('p', gelu='relu', **formats)                 # also where an engine is there already
    again = M.MI355XRuntime('p', gelu='erf', reload=True, **formats)
    assert again.engine is not erf.engine and not again.engine.gelu_tanh and len(loads) == 3


def test_formats_and_paths_are_kept_apart(loads):
    a = M.MI355XRuntime('p', decoder_format='mxfp4')
    b = M.MI355XRuntime('p', encoder_mlp_format='mxfp4')
    c, d = M.MI355XRuntime('p'), M.MI355XRuntime('q', decoder_format='mxfp4')
    assert len({id(r.engine) for r in (a, b, c, d)}) == 4 == len(loads)


@pytest.mark.parametrize('formats', [{}, dict(decoder_format='mxfp4')])
def test_an_engine_asked_for_in_one_form_is_not_the_default(loads, formats):
    erf = M.MI355XRuntime('p', gelu='erf', **formats)
    assert M.MI355XRuntime('p', **formats).engine.gelu_tanh and not erf.engine.gelu_tanh


def test_a_reload_leaves_no_older_engine_behind(loads):
    old = M.MI355XRuntime('p').engine
    assert M.MI355XRuntime('p', gelu='tanh').engine is old
    erf = M.MI355XRuntime('p', gelu='erf').engine
    new = M.MI355XRuntime('p', reload=True).engine
    assert new is not old and M.MI355XRuntime('p', gelu='tanh').engine is new
    assert M.MI355XRuntime('p', gelu='erf').engine is not erf


def test_options_that_a_given_engine_does_not_have_are_refused(loads):
    plain = M.MI355XRuntime('p').engine
    four = M.MI355XRuntime('p', decoder_format='mxfp4').engine
    for engine, options in ((plain, dict(decoder_format='mxfp4')), (plain, dict(encoder_mlp_format='mxfp4')), (four, dict(encoder_mlp_format='mxfp4')),
                            (four, dict(decoder_format='int8')), (plain, dict(gelu='erf')), (plain, dict(gelu='relu'))):
        with pytest.raises(ValueError):
            M.MI355XRuntime('p', engine=engine, **options)
    for engine, options in ((plain, {}), (four, {}), (four, dict(decoder_format='mxfp4')), (plain, dict(gelu='tanh'))):
        assert M.MI355XRuntime('p', engine=engine, **options).engine is engine
    assert len(loads) == 2
    erf = M.MI355XRuntime('p', gelu='erf').engine
    with pytest.raises(ValueError):
        M.MI355XRuntime('p', engine=erf, gelu='relu')
