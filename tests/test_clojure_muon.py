"""What the text of the Clojure optimizer for matrices has to say, since no JVM is here to run it: a network hands every parameter to one
optimizer, so what is no matrix goes to another one, which is also told of each batch; matrices of experts go to the step together."""
from test_clojure_glue import GLUE, read_forms, walk

FORMS = read_forms(next(p for p in GLUE if p.name == "optimize.clj").read_text())


def form(*start):
    return next(f for f in walk(FORMS) if f[1:1 + len(start)] == list(start))


def test_parameters_that_are_no_matrices_take_another_optimizers_step():
    record = form("defrecord", "HipMuon")
    method = next(f for f in walk(record) if f[1:2] == ["compute-parameters!"] and "state" in str(f[2]))
    choice = next(f for f in walk(method) if f[1:2] == ["if-not"])
    assert choice[2][1:] == ["<=", "2", ["(", "count", "shape"], "3"]
    assert choice[3][1:] == ["compute-parameters!", "vectors", "state", "gradient-alpha", "offset", "gradient", "parameters"]
    assert not any(f[1:2] == ["throw"] for f in walk(method))
    told = next(f for f in walk(record) if f[1:2] == ["batch-update"] and f is not record)
    assert ["(", "batch-update", "%", "optimizer-parameters"] in list(walk(told))


def test_matrices_of_experts_and_coefficients_of_each_step():
    step = next(f for f in walk(form("defrecord", "HipMuon")) if f[1:2] == ["call!"])
    assert step[2] == ("str", "ct_muon_step")
    assert ["(", "long", "n-matrices"] in step
    triples = form("defn-", "steps->triples")
    assert ["(", "number?", ["(", "first", "coefficients"]] in list(walk(triples)) and any(f[1:2] == ["throw"] for f in walk(triples))
