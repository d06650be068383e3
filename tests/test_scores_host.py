"""What tgbm_scores_* refuse is refused before anything reaches a GPU: the pointers here are never followed."""
import ctypes as C

import pytest

P = 1 << 20   # an address that is aligned for everything


@pytest.fixture(scope='module')
def lib():
    from thundergbm_b200 import _lib
    return _lib.lib()


def _adjust(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, out=P + 65536, ors=40, ocs=1, bias=None, allowed=None, masks=0, words=0, row=None, ptr=None, ids=None,
            given=0, r=1.0, f=0.0, p=0.0):
    return lib.tgbm_scores_adjust(n, k, type, z, rs, cs, out, ors, ocs, bias, allowed, masks, words, row, ptr, ids, given, r, f, p, None)


def _top(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, m=3, T=1.0, v=P, i=P, lse=None):
    return lib.tgbm_scores_top(n, k, type, z, rs, cs, m, T, v, i, lse, None)


def _distill(lib, n=4, k=40, type=0, z=P, rs=40, cs=1, m=3, ids=P, ids_stride=3, lt=0, logits=P, logits_stride=3, T=1.0, a=1.0, loss=P, gives=1, g=P + 65536, grs=40,
             gcs=1):
    return lib.tgbm_scores_distill(n, k, type, z, rs, cs, m, ids, ids_stride, lt, logits, logits_stride, None, None, None, T, a, loss, gives, g, grs, gcs, None)


NAN, INF = float('nan'), float('inf')


@pytest.mark.parametrize('call,args,says', [
    (_adjust, dict(n=-1), 'rows'), (_adjust, dict(k=0), 'classes'), (_adjust, dict(k=(1 << 20) + 1), 'classes'), (_adjust, dict(type=3), 'type'),
    (_adjust, dict(z=None), 'null'), (_adjust, dict(z=P + 2), 'aligned'), (_adjust, dict(rs=-40), 'negative'), (_adjust, dict(cs=1 << 62), 'large'),
    (_adjust, dict(ors=39), 'share'), (_adjust, dict(ocs=0), 'share'), (_adjust, dict(out=P + 4), 'share'), (_adjust, dict(out=P, ors=80), 'share'),
    (_adjust, dict(out=P + 160 * 2), 'share'), (_adjust, dict(r=0.0), 'repetition'), (_adjust, dict(r=NAN), 'repetition'), (_adjust, dict(f=INF), 'finite'),
    (_adjust, dict(allowed=P, masks=0, words=2), 'masks'), (_adjust, dict(allowed=P, masks=4, words=1), 'shorter'),
    (_adjust, dict(allowed=P, masks=3, words=2), 'fewer'), (_adjust, dict(given=-1), 'negative'), (_adjust, dict(ptr=P, given=5), 'history'),
    (_top, dict(m=0), 'list'), (_top, dict(m=129), 'list'), (_top, dict(T=0.0), 'temperature'), (_top, dict(T=INF), 'temperature'), (_top, dict(T=NAN), 'temperature'),
    (_top, dict(T=1e-40), 'temperature'), (_top, dict(v=None), 'null'), (_top, dict(i=None), 'null'), (_top, dict(type=-1), 'type'), (_top, dict(n=-5), 'rows'),
    (_distill, dict(m=200), 'list'), (_distill, dict(a=-0.1), 'alpha'), (_distill, dict(a=NAN), 'alpha'), (_distill, dict(gives=3), 'kind'), (_distill, dict(lt=9), 'logits'),
    (_distill, dict(ids=None), 'null'), (_distill, dict(logits=None), 'null'), (_distill, dict(ids_stride=-1), 'negative'), (_distill, dict(gives=0, loss=None), 'loss'),
    (_distill, dict(g=None), 'null'), (_distill, dict(gives=2, g=P + 65540), 'aligned'), (_distill, dict(g=P), 'share'), (_distill, dict(grs=1, gcs=1), 'share'),
    (_distill, dict(gives=2, g=P + 8), 'share'),
    (_adjust, dict(bias=P + 2), 'aligned'), (_adjust, dict(ptr=P + 4, ids=P, given=5), 'aligned'), (_top, dict(v=P + 1), 'aligned'), (_distill, dict(ids=P + 2), 'aligned'),
    (_distill, dict(lt=0, logits=P + 2), 'aligned'), (_distill, dict(loss=P + 3), 'aligned'),
])
def test_refused(lib, call, args, says):
    assert call(lib, **args) == 1
    assert says in lib.tgbm_last_error().decode()


@pytest.mark.parametrize('call', [_adjust, _top, _distill])
def test_no_rows_is_nothing_to_do(lib, call):
    assert call(lib, n=0, z=None) == 0
    assert lib.tgbm_last_error() == b''


@pytest.mark.parametrize('r', [1e-40, 2.9e-39, 1e-45])
def test_a_repetition_penalty_without_a_reciprocal_is_refused(lib, r):
    """Scores are divided through the penalty's reciprocal, which a float has to hold: 1e-5 / 1e-40 is one, 1 / 1e-40 is not."""
    assert _adjust(lib, r=r) == 1
    assert 'repetition' in lib.tgbm_last_error().decode()


FAR = 1 << 30


@pytest.mark.parametrize('call,args', [
    # out is 4 x 40 floats, 640 bytes, at P + 65536; what is read begins or ends inside
    (_adjust, dict(bias=P + 65536)), (_adjust, dict(bias=P + 65536 - 156)), (_adjust, dict(bias=P + 65536 + 636)),
    (_adjust, dict(allowed=P + 65536 - 28, masks=4, words=2)), (_adjust, dict(allowed=FAR, masks=4, words=2, row=P + 65536 + 600)),
    (_adjust, dict(ptr=P + 65536 - 32, ids=FAR, given=5)), (_adjust, dict(ptr=FAR, ids=P + 65536 - 16, given=5)),
    (_adjust, dict(out=P, bias=P + 160)),   # in place, with a row of the scores as a bias
])
def test_results_over_what_is_read_are_refused(lib, call, args):
    assert call(lib, **args) == 1
    assert 'share memory' in lib.tgbm_last_error().decode()


@pytest.mark.parametrize('call', [_top, _distill])
@pytest.mark.parametrize('T', [3e-39, 4.2e-39])
def test_temperatures_whose_exponents_no_float_holds_are_refused(lib, call, T):
    """exp(x / T) is 2^(x log2(e) / T): a float has to hold log2(e) / T, not only 1 / T."""
    assert call(lib, T=T, **({'logits': P + 4096} if call is _distill else {})) == 1
    assert 'temperature' in lib.tgbm_last_error().decode()
