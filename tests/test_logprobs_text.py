"""Log probabilities of completions and the response's text: where tokens begin in it, characters in several tokens, special tokens (CPU)."""
import codecs
import json
import random

import pytest

from b200serve.server.app import Server, ServerOptions
from b200serve.server.chat_template import ChatTemplate
from b200serve.server.iface import ByteTok, MockEngine, NativeTok
from b200serve.server.logprobs import Entry, Place, Score, text_block
from test_server import TOK, enc, post

V = 259


@pytest.fixture()
def serve():
    servers = []

    def make(script, tok=TOK, vocab=V, **kw):
        srv = Server(MockEngine(vocab_size=vocab, max_len=2048, max_seqs=2, script=script), tok, ChatTemplate(), ServerOptions(**kw)).start()
        servers.append(srv)
        return srv
    yield make
    for s in servers:
        s.stop()


def complete(srv, stream, **body):
    """(text, the blocks of log probabilities joined)."""
    body["stream"] = stream
    if not stream:
        ch = post(srv.port, "/v1/completions", body)[1]["choices"][0]
        return ch["text"], ch["logprobs"]
    ch = [json.loads(f)["choices"][0] for f in post(srv.port, "/v1/completions", body, stream=True)[1][:-1]]
    blocks = [c["logprobs"] for c in ch if c.get("logprobs")]
    return "".join(c["text"] for c in ch), {k: sum((b[k] or [] for b in blocks), []) for k in blocks[0]}


def byte_places(text):
    """Of every byte of a text's UTF-8 form: the place of the character that it belongs to."""
    return [i for i, c in enumerate(text) for _ in c.encode()]


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("text", ["été x", "日本 a語", "a😀b", "ü"])
def test_offsets_of_characters_in_several_tokens(serve, stream, text):
    srv = serve({enc("go "): list(enc(text))})
    out, lp = complete(srv, stream, prompt="go ", max_tokens=len(enc(text)), logprobs=1)
    assert out == text and lp["text_offset"] == byte_places(text)
    for token, at in zip(lp["tokens"], lp["text_offset"]):
        if len(token) == 1 and token.isascii():
            assert out[at:].startswith(token)


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("as_ids", [False, True])
def test_offsets_behind_an_echoed_prompt(serve, stream, as_ids):
    text, more = "né 日", "ö!"
    srv = serve({enc(text): list(enc(more))})
    out, lp = complete(srv, stream, prompt=list(enc(text)) if as_ids else text, max_tokens=len(enc(more)), logprobs=0, echo=True)
    assert out == text + more and lp["text_offset"] == byte_places(text + more)


def test_a_prompt_that_ends_inside_a_character(serve):
    """The prompt's text and the completion's are decoded each for itself: half a character at the end of the one, half at the beginning of the other."""
    ids = list(enc("aé"))
    srv = serve({tuple(ids[:2]): [ids[2]] + list(enc("b"))})
    out, lp = complete(srv, False, prompt=ids[:2], max_tokens=2, logprobs=0, echo=True)
    assert out == "a��b" and lp["text_offset"] == [0, 1, 2, 3]


def test_special_tokens_take_no_place_where_the_text_leaves_them_out(serve):
    a, b, c = (enc(x)[0] for x in "abc")
    srv = serve({(1, a, 1, b): [1, c, 0, a]})
    out, lp = complete(srv, False, prompt=[1, a, 1, b], max_tokens=4, logprobs=0, echo=True)
    assert out == "abca" and lp["text_offset"] == [0, 0, 1, 1, 2, 2, 3, 3]


@pytest.fixture()
def native(tmp_path):
    """Byte-level tokens, one of two bytes, one special and one added token."""
    vocab, n = {}, 0
    for v in range(256):      # the usual names of bytes
        keep = 33 <= v <= 126 or 161 <= v <= 172 or 174 <= v <= 255
        vocab[chr(v if keep else 256 + n)] = v
        n += not keep
    vocab["he"] = 256
    spec = {"model": {"vocab": vocab, "merges": ["h e"]}, "added_tokens": [{"content": "<|bos|>", "id": 257, "special": True}, {"content": "<tool>", "id": 258, "special": False}]}
    path = tmp_path / "tokenizer.json"
    path.write_text(json.dumps(spec))
    return NativeTok(str(path))


def test_text_bytes_are_what_the_text_gains(native):
    assert native.text_bytes(257) == b"" and native.token_bytes(257) == b"<|bos|>" and native.text_bytes(258) == b"<tool>" and native.text_bytes(256) == b"he"
    for ids in ([257, 256, 258, 195, 169], [256, 257]):
        s = native.streamer()
        assert b"".join(bytes(s.push(i)) for i in ids) + bytes(s.finish()) == b"".join(native.text_bytes(i) for i in ids) == native.decode(ids).encode()


@pytest.mark.parametrize("stream", [False, True])
def test_special_tokens_of_a_prompt_stand_in_its_own_text(serve, native, stream):
    ids = native.encode("<|bos|>hé<tool>x")
    assert ids == [257, 104, 195, 169, 258, 120]
    srv = serve({tuple(ids): [257, 104, 105]}, tok=native)
    out, lp = complete(srv, stream, prompt="<|bos|>hé<tool>x", max_tokens=3, logprobs=0, echo=True)
    assert out == "<|bos|>hé<tool>xhi" and lp["text_offset"] == [0, 7, 8, 8, 9, 15, 16, 16, 17]
    out, lp = complete(srv, stream, prompt=ids, max_tokens=3, logprobs=0, echo=True)
    assert out == "hé<tool>xhi" and lp["text_offset"] == [0, 0, 1, 1, 2, 8, 9, 9, 10]


def char_ends(raw):
    """The byte behind each character of a text decoded as a whole, replacement characters among them."""
    bad = []

    def note(e):
        bad.append((e.start, e.end))
        return "\ufffd", e.end
    codecs.register_error("note", note)
    raw.decode("utf-8", "note")
    ends, at = [], 0
    for lo, hi in bad + [(len(raw), len(raw))]:
        for ch in raw[at:lo].decode():
            at += len(ch.encode())
            ends.append(at)
        if hi > lo:
            ends.append(hi)
        at = hi
    return ends


def test_bytes_that_are_no_text():
    """Against the whole text decoded at once: a token's place is the number of characters that end before its first byte."""
    rnd = random.Random(3)
    pieces = ["a", "é", "日", "😀"]
    for _ in range(400):
        raw = b"".join(rnd.choice([rnd.choice(pieces).encode(), bytes([rnd.randrange(256)]), rnd.choice(pieces).encode()[:-1]]) for _ in range(12))
        ends, place, i = char_ends(raw), Place(), 0
        assert len(ends) == len(raw.decode("utf-8", "replace"))
        while i < len(raw):
            n = rnd.randrange(1, 4)
            assert place.add(raw[i: i + n]) == sum(e <= i for e in ends), (raw, i)
            i += n
        assert place.at + len(place.held.decode("utf-8", "replace")) == len(ends)


def test_blocks_that_begin_somewhere():
    e = [Entry(t, Score(-1.0, [])) for t in enc("é!")]
    block, at = text_block(ByteTok(), e, 0, 4)
    assert block["text_offset"] == [4, 4, 5] and at == 6
    block, _ = text_block(ByteTok(), [Entry(enc("x")[0], None, 9), Entry(enc("y")[0], None, 3)], 0, 0)
    assert block["text_offset"] == [9, 3]


def test_alternatives_that_are_parts_of_characters():
    """Tokens that are no text by themselves are told apart, and the token itself keeps its own number."""
    a, b, c = enc("é日")[:3]
    block, _ = text_block(TOK, [Entry(a, Score(-3.0, [(b, -0.5), (c, -1.0)])), Entry(b, Score(-3.25, [(c, -0.5)]))], 2, 0)
    assert block["tokens"] == ["bytes:\\xc3", "bytes:\\xa9"]
    assert block["top_logprobs"] == [{"bytes:\\xc3": -3.0, "bytes:\\xa9": -0.5, "bytes:\\xe6": -1.0}, {"bytes:\\xa9": -3.25, "bytes:\\xe6": -0.5}]
    # an alternative of the same text (ids 0 and 1 have none): the token's own number
    block, _ = text_block(TOK, [Entry(1, Score(-4.0, [(0, -0.25), (a, -2.0)]))], 2, 0)
    assert block["top_logprobs"] == [{"": -4.0, "bytes:\\xc3": -2.0}]


@pytest.mark.parametrize("stream", [False, True])
def test_every_token_is_among_its_alternatives(serve, stream):
    srv = serve({enc("go "): list(enc("日é"))})
    out, lp = complete(srv, stream, prompt="go ", max_tokens=5, logprobs=2)
    assert out == "日é" and len(lp["tokens"]) == 5
    for token, number, top in zip(lp["tokens"], lp["token_logprobs"], lp["top_logprobs"]):
        assert len(top) == 2 and top[token] == number == max(top.values())
