"""Recognizer shell with the reference's constructor wiring (lnasr/recognizer.py:20-48).

The reference's `recognize()` is unimplemented (`pass`) and its language-model / lexicon side
is out of scope here.  `AcousticModel` wires MFCC + GMMHMM exactly as the
reference does; `Recognizer.recognize` runs the acoustic path the reference stops short of:
PCM -> MFCC -> Viterbi state path.  Upstream has nothing to compare with; the checker is the composition of the two
oracle-pinned halves, oracle.mfcc -> oracle.decode (tests/test_gpu_frontend.py::test_recognize_equals_oracle_chain).
The samples go to the device once; features, emissions and trellis stay in HBM and only the path [Nf] comes back.
"""
import numpy as np

from .mfcc import MFCC
from .gmmhmm import GMMHMM
from .transform import SpeakerTransforms


class AcousticModel:
    def __init__(self, modelfile):
        self.mfcc = MFCC()
        self.gmmhmm = GMMHMM(n=2, m=2, d=self.mfcc.D)
        self.gmmhmm.load(modelfile)


class LanguageModel:
    """The n-gram language model is not part of the accelerated path; the model file is only recorded."""

    def __init__(self, modelfile):
        self.modelfile = modelfile
        self.ngram = None


class Recognizer:
    def __init__(self, model: dict):
        self.am = AcousticModel(model["am"])
        self.lm = LanguageModel(model["lm"]) if model.get("lm") is not None else None
        # "transform" (an extension): a file of SpeakerTransforms, applied between MFCC and decoding
        self.transforms = None
        if model.get("transform") is not None:
            self.transforms = SpeakerTransforms()
            self.transforms.load(model["transform"])

    def recognize(self, data: np.ndarray, speaker=0):
        """PCM samples (int16 as read_pcm returns them, utils.py:100-104, or float64) -> most likely HMM state sequence
        (uint32 [Nf]).  speaker: whose transform the features take, where the model has transforms."""
        data = np.ascontiguousarray(data)
        if data.dtype != np.int16:
            data = np.ascontiguousarray(data, dtype=np.float64)
        mf, gh = self.am.mfcc, self.am.gmmhmm
        ctx = gh.ctx
        cfg, win, bank = mf._cfg()
        d_pcm = ctx.to_device(data)
        _, _, feat, _ = ctx.mfcc(d_pcm, np.array([0, len(data)], dtype=np.int64), cfg, win, bank, False, False)
        if self.transforms is not None:
            feat = self.transforms.apply(feat, np.array([0, feat.shape[0]], dtype=np.int64), np.array([speaker]))
        return gh.decode(feat)

    def recognize_batch(self, utterances, speakers=None):
        """Many utterances at once (all int16, or float64) -> a list of state sequences.  speakers: the speaker of each, where the
        model has transforms (default: speaker 0).  Features, transforms, emissions and trellises stay in HBM."""
        utterances = [np.asarray(u) for u in utterances]
        if not utterances:
            return []
        dt = np.int16 if all(u.dtype == np.int16 for u in utterances) else np.float64
        mf, gh = self.am.mfcc, self.am.gmmhmm
        ctx = gh.ctx
        cfg, win, bank = mf._cfg()
        offsets = np.concatenate([[0], np.cumsum([len(u) for u in utterances])]).astype(np.int64)
        d_pcm = ctx.to_device(np.concatenate(utterances).astype(dt))
        _, _, feat, rows = ctx.mfcc(d_pcm, offsets, cfg, win, bank, False, False)
        if self.transforms is not None:
            speakers = np.zeros(len(utterances), dtype=np.int32) if speakers is None else np.asarray(speakers)
            feat = self.transforms.apply(feat, rows, speakers)
        obs, lens = ctx.pad_rows(feat, rows)
        gh.upload()
        path = gh.decode_batch(obs, lens=lens).to_host()
        return [path[u, :n] for u, n in enumerate(lens)]
